// Choosing the next token from a row of logits and given random numbers.
//
// With best = max l, x_i = (l_i - best) / T and w_i = exp(x_i), the tokens in falling order of their
// logit (the lower index first among equals) are cut to a prefix twice: to the first top_k, and to
// those before whom less than top_p of that prefix's mass lies; tokens with w_i < min_p leave too.
// The first token always stays.  Of what is left the token with the largest w_i / e_i is taken (the
// lowest index among equals): with e_i independent and exponentially distributed that is a draw from
// the softmax of what is left, and unlike a walk along the cumulative sum it compares single numbers,
// so the rounding of a long sum never decides it.  T <= 0 takes the first token.  The second result is
// the token's log-probability under the whole row at this temperature (1 where T <= 0).
// Logits of -inf or NaN cannot be drawn; a row without any other gives token -1 and -inf.
//
// Bound: memory (the logits once, and the random numbers of the tokens that may be drawn); at a handful of
// rows, the latency of the steps.  A row belongs to a cluster of blocks, which exchange a few numbers per step
// through distributed shared memory.  (Many rows of which nothing is cut are streamed by another kernel, see `streams`.)  There
// are three ways through a row, each with fewer steps than the next:
//
// * Nothing to cut (no top_k, top_p or min_p, or T <= 0): one pass over logits and random numbers with a running
//   reference for the exponentials, rescaled by powers of two, so that no step waits for the maximum.
// * Short prefix: the row is held in shared memory.  The median of the warps' largest logits is a threshold that
//   some 100 tokens reach, whatever the distribution; they are sent to the first block, which ranks them against
//   one another, cuts and draws.  Taken when those tokens provably hold both cuts; otherwise
// * a lower threshold of the same kind, that some 1500 tokens reach, is tried, and then all tokens: a cut is found
//   without sorting from a histogram over 2048 bins of falling logit, of counts for top_k and of masses for
//   top_p.  The one bin that holds the boundary is resolved: its tokens are ranked against one another, or, if
//   there are many, divided further by their bits (those of the index below those of the logit, so that equal
//   logits divide too).  The first block does that for the 1500, the cluster for all.
//
// Masses are integers, round(w 2^44) of up to 2^18 tokens in 64 bits.  Integer sums do not depend on their order, so neither do
// the cuts.  The histograms hold 31 bits of a weight, split into halves of 16 bits that 32-bit shared-memory atomics add without
// overflow, in units that go with the bin (a bin's weights differ by a factor of e^(1/64)) down to 2^-44, so that a share near 1
// is cut where the sum says: with multiples of 2^-31 for all, a tail of 128256 tokens of 2^-30 was off by 1e-5 of the whole.
// (256 rows at T = 1.3 with top-p 0.95: 458 us, 455 without.)
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "sampling.cuh"

namespace cg = cooperative_groups;

namespace ht {
namespace sampling {

constexpr int BINS = 2048;
constexpr int LIST = 256;       // tokens of one bin that are ranked directly
constexpr int SHORT = 256;      // tokens of a short prefix
constexpr int MEDIUM = 2048;    // tokens of a longer one, or of one bin
constexpr int STAGED = BINS * 3 / 2;  // tokens that the bins' memory holds
constexpr int MOST_BLOCKS = 8;  // of a cluster

struct Found {  // where a running sum over the bins crosses its target
  int bin;
  uint32_t count;            // tokens of the bin
  unsigned long long before;  // sum of the bins in front of it
};

struct Warp {
  float reference;
  double sum;
  unsigned long long pick;
};

struct Shared {
  Warp warps[MOST_BLOCKS][WARPS];
  uint32_t warp_top[2][WARPS];
  bool fine;
  alignas(8) uint32_t count[BINS], low[BINS], high[BINS];  // masses: 2^16 high + low, in the bin's units; between uses, what `gather` collects
  unsigned long long list[MEDIUM], bin_list[LIST];
  unsigned long long list_mass[SHORT];
  uint32_t bin_mass[LIST];
  uint32_t listed, bin_listed, staged, room;
  unsigned long long scan[WARPS];
  uint32_t reduce32[WARPS];
  unsigned long long slice[MOST_BLOCKS];                      // per block of the cluster
  uint32_t keys[3][MOST_BLOCKS];                              // likewise
  unsigned long long ends[2][MOST_BLOCKS];                    // likewise
  double totals[MOST_BLOCKS], reduce64[WARPS];                // likewise
  unsigned long long masses[MOST_BLOCKS];                     // likewise
  uint32_t counts[MOST_BLOCKS];                               // likewise
  Found found;
  unsigned long long cut;
};

// Bins of 1/64 of the exponent (to base e) for the first 32; everything further away shares the last bin.  Monotone in l,
// as every step of its computation is.
__device__ __forceinline__ int first_bin(const Weights& weight, float l) {
  return (int)fminf(weight.exponent(l) * (-64.f * LN2), (float)(BINS - 1));
}

// Weights of such a bin are at most 2^-k, k = floor(bin / 64 log2(e)); bins hold them in multiples of 2^-(31 + k), down to 2^-44.
__device__ __forceinline__ int bin_power(int bin) { return min(bin * 1477 >> 16, 13); }

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const __grid_constant__ Args a) {
  constexpr int E = Piece<T>::E;
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  uint4* const held = reinterpret_cast<uint4*>(smem + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / blocks, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const auto peer = [&](auto* p, int r) { return cluster.map_shared_rank(p, r); };

  const float temperature = a.temperature[row];
  const bool greedy = !(temperature > 0.f);
  const int top_k = a.top_k[row];
  // A NaN as top_p or min_p keeps the most probable token alone: its share is a mass of 1, and no weight is at or above it.
  const float top_p = a.top_p[row], min_p = a.min_p[row];
  // This launch may begin before the streaming one, whose results it does not read, has ended; it must not end before that one.
  if (a.streamed && row == a.B - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (a.streamed && ordinary(temperature) && cuts_nothing(top_k, top_p, min_p, a.V)) return;
  // Shared memory of a peer may be written once that block runs.  Every thread announces itself here and asks once, before the
  // first exchange; the row's loads lie between.
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  bool asked = false;
  const auto peers_run = [&] {
    if (!asked) asm volatile("barrier.cluster.wait;" ::: "memory");
    asked = true;
  };
  const bool by_count = !greedy && top_k > 0 && top_k < a.V, by_mass = !greedy && !(top_p >= 1.f);
  const float* const noise = a.noise + row * a.noise_stride;

  // ---- this block's stretch of the row, as aligned pieces of 16 bytes; places outside the row hold -inf
  const T* const logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(logits) % 16) / sizeof(T));
  const uint4* const aligned = reinterpret_cast<const uint4*>(logits - skew);
  const int pieces = (skew + a.V + E - 1) / E, each = (pieces + blocks - 1) / blocks;
  const int from = min(rank * each, pieces), count = min(each, pieces - from);
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  // A token outside the row's ends may not be read: f(index in the piece, token) for those inside.
  const auto inside = [&](int i) {  // whether all of the piece belongs to the row
    const int first = (from + i) * E - skew;
    return first >= 0 && first + E <= a.V;
  };
  const auto end_piece = [&](int i) {  // a piece at one of the row's ends
    uint32_t u[4] = {none, none, none, none};
    for (int e = 0; e < E; ++e) {
      const int token = (from + i) * E - skew + e;
      if (token < 0 || token >= a.V) continue;
      if constexpr (sizeof(T) == 4) u[e] = __float_as_uint(logits[token]);
      else u[e / 2] = (u[e / 2] & (e % 2 ? 0xffffu : 0xffff0000u)) | ((uint32_t)__bfloat16_as_ushort(logits[token]) << (16 * (e % 2)));
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  };
  const auto better = [](unsigned long long x, unsigned long long y) { return x > y ? x : y; };

  // ---- one pass, where nothing is cut and the temperature is an ordinary one
  if (!by_count && !by_mass && (greedy || (min_p <= 0.f && temperature > 1e-3f && temperature < 1e3f))) {
    const double rate = 1.4426950408889634 / (greedy ? 1.0 : (double)temperature);
    const float hi = (float)rate, lo = (float)(rate - (double)hi);
    const bool together = (reinterpret_cast<uintptr_t>(noise - skew) % 16) == 0;
    constexpr int DEPTH = E == 4 ? 8 : 4;  // pieces of a thread in flight: 128 bytes of random numbers
    float reference = -1e30f, best = greedy ? -INFINITY : -1.f, sum = 0.f;  // exponents are taken from `reference`, an integer
    int winner = a.V;
    for (int i0 = tid; i0 < count; i0 += DEPTH * THREADS) {
      // all of the turn is under way before its first half is used: logits to shared memory, random numbers to registers
      float4 luck[DEPTH][E / 4];
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        const int i = i0 + j * THREADS;
        if (i < count && inside(i)) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(held + i)), "l"(aligned + from + i) : "memory");
          if (!greedy && together) {
#pragma unroll
            for (int x = 0; x < E / 4; ++x) luck[j][x] = __ldcs(reinterpret_cast<const float4*>(noise + (from + i) * E - skew) + x);
          }
        }
        if (j == DEPTH / 2 - 1) asm volatile("cp.async.commit_group;" ::: "memory");
      }
      asm volatile("cp.async.commit_group;\n cp.async.wait_group 1;" ::: "memory");  // a thread reads what it copied itself
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        if (j == DEPTH / 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
        const int i = i0 + j * THREADS, first = (from + i) * E - skew;
        if (i >= count) continue;
        Piece<T> p(inside(i) ? held[i] : end_piece(i));
        if (!greedy && !(together && inside(i))) {
          float* const e = reinterpret_cast<float*>(luck[j]);
#pragma unroll
          for (int x = 0; x < E; ++x) e[x] = first + x >= 0 && first + x < a.V ? noise[first + x] : 1.f;
        }
        float top = -1e30f;
#pragma unroll
        for (int x = 0; x < E; ++x) {
          p.v[x] = fmaxf(p.v[x], -1e30f);  // -inf and NaN: no weight at any ordinary temperature
          top = fmaxf(top, p.v[x]);
        }
        if (!(top > -1e30f)) continue;  // nothing to draw here
        if (top * hi > reference) {
          const float higher = ceilf(top * hi), scale = fast_exp2(reference - higher);
          sum *= scale;
          if (!greedy && best > 0.f) best *= scale;
          reference = higher;
        }
#pragma unroll
        for (int x = 0; x < E; ++x) {
          const float w = fast_exp2(fmaf(p.v[x], lo, fmaf(p.v[x], hi, -reference)));
          sum += w;
          // a NaN (from a random number that is none) loses to every score, but still names a token
          const float score =
              greedy ? p.v[x] : p.v[x] > -1e30f ? fmaxf(__fdividef(w, reinterpret_cast<const float*>(luck[j])[x]), -0.5f) : -1.f;
          if (score > best) {
            best = score;
            winner = first + x;
          }
        }
      }
    }
    float highest = reference;
    for (int o = 16; o > 0; o >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, o));
    const float scale = fast_exp2(reference - highest);
    if (!greedy && best > 0.f) best *= scale;
    double of_warp = (double)(sum * scale);
    unsigned long long pick = ((unsigned long long)key_of(best) << 32) | (0xffffffffu - (uint32_t)winner);
    for (int o = 16; o > 0; o >>= 1) {
      of_warp += __shfl_xor_sync(0xffffffffu, of_warp, o);
      pick = better(pick, __shfl_xor_sync(0xffffffffu, pick, o));
    }
    // every warp sends its three numbers to every block, which come to the same conclusion
    peers_run();
    if (lane < blocks) {
      Warp& to = *peer(&sh.warps[rank][warp], lane);
      to.reference = highest;
      to.sum = of_warp;
      to.pick = pick;
    }
    cluster.sync();
    const int n = blocks * WARPS;
    if (warp == 0) {
      const Warp* const all = &sh.warps[0][0];
      float most = -INFINITY;
      for (int i = lane; i < n; i += 32) most = fmaxf(most, all[i].reference);
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      // beyond this the products with the rate lose the differences (or a logit is infinite): the row is held instead
      const bool fine = fabsf(most) < 1e5f;
      double whole = 0.0;
      unsigned long long choice = 0;
      for (int i = lane; i < n; i += 32) {
        const float down = fast_exp2(all[i].reference - most);
        whole += all[i].sum * (double)down;
        const uint32_t key = (uint32_t)(all[i].pick >> 32);
        const float score = value_of(key);
        choice = better(choice, greedy || !(score > 0.f) ? all[i].pick
                                                        : ((unsigned long long)key_of(score * down) << 32) | (uint32_t)all[i].pick);
      }
      for (int o = 16; o > 0; o >>= 1) {
        whole += __shfl_xor_sync(0xffffffffu, whole, o);
        choice = better(choice, __shfl_xor_sync(0xffffffffu, choice, o));
      }
      if (lane == 0) {
        sh.fine = fine;
        if (fine && rank == 0) {
          const int token = (int)(0xffffffffu - (uint32_t)choice);
          const float l = Piece<T>::one(logits[token]);
          a.token[row] = token;
          a.logprob[row] = (fmaf(l, lo, fmaf(l, hi, -most)) - __log2f((float)whole)) * LN2;
        }
      }
    }
    __syncthreads();
    if (sh.fine) return;
  }

  float top = -INFINITY;  // of the thread's own pieces
  const auto keep_piece = [&](int i, uint4 raw) {
    uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    Piece<T> p(raw);
    bool odd = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      odd |= p.v[e] != p.v[e];
      top = fmaxf(top, p.v[e]);
    }
    if (odd) {  // NaN becomes -inf
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          if (p.v[j] != p.v[j]) u[j] = none;
        } else {
          if (p.v[2 * j] != p.v[2 * j]) u[j] = (u[j] & 0xffff0000u) | (none & 0xffffu);
          if (p.v[2 * j + 1] != p.v[2 * j + 1]) u[j] = (u[j] & 0xffffu) | (none & 0xffff0000u);
        }
      }
    }
    held[i] = make_uint4(u[0], u[1], u[2], u[3]);
  };
  {
    constexpr int DEPTH = 4;
    for (int i0 = tid; i0 < count; i0 += DEPTH * THREADS) {
      uint4 raw[DEPTH];
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        const int i = i0 + j * THREADS;
        raw[j] = make_uint4(none, none, none, none);
        if (i < count && inside(i)) raw[j] = __ldcs(aligned + from + i);
      }
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        const int i = i0 + j * THREADS;
        if (i >= count) continue;
        if (!inside(i)) raw[j] = end_piece(i);
        keep_piece(i, raw[j]);
      }
    }
  }
  const uint32_t own_top = key_of(top);
  // The block's largest key, and two thresholds: the medians over its warps of the largest keys of their lanes' (in smaller
  // clusters the second, fourth or eighth largest), and of the tenth largest (in smaller clusters lower ones, so that
  // the number of tokens above it stays).  Some tokens of every block reach the lowest of the blocks' medians.
  uint32_t best_key = 0, threshold = 0xffffffffu, lower = 0xffffffffu;
  {
    int above = 0;
#pragma unroll 8
    for (int x = 0; x < 32; ++x) {
      const uint32_t other = __shfl_sync(0xffffffffu, own_top, x);
      above += other > own_top || (other == own_top && x < lane);
    }
    if (above == 0) sh.reduce32[warp] = own_top;
    if (above == MOST_BLOCKS / blocks - 1) sh.warp_top[0][warp] = own_top;
    if (above == (blocks == 8 ? 9 : blocks == 4 ? 15 : blocks == 2 ? 23 : 29)) sh.warp_top[1][warp] = own_top;
    if (tid == 0) sh.listed = sh.bin_listed = 0u;
    __syncthreads();
    peers_run();
    if (warp == 0) {
      uint32_t medians[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t mine = lane < WARPS ? sh.warp_top[y][lane] : 0u;
        int higher = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const uint32_t other = __shfl_sync(0xffffffffu, mine, w);
          higher += other > mine || (other == mine && w < lane);
        }
        medians[y] = __reduce_max_sync(0xffffffffu, lane < WARPS && higher == WARPS / 2 - 1 ? mine : 0u);
      }
      const uint32_t most = __reduce_max_sync(0xffffffffu, lane < WARPS ? sh.reduce32[lane] : 0u);
      if (lane < blocks) {
        *peer(&sh.keys[0][rank], lane) = most;
        *peer(&sh.keys[1][rank], lane) = medians[0];
        *peer(&sh.keys[2][rank], lane) = medians[1];
      }
    }
    cluster.sync();
    for (int r = 0; r < blocks; ++r) {
      best_key = max(best_key, sh.keys[0][r]);
      threshold = min(threshold, sh.keys[1][r]);
      lower = min(lower, sh.keys[2][r]);
    }
  }
  if (best_key == 0u) {  // the same for every block of the cluster
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      a.logprob[row] = -INFINITY;
    }
    return;
  }

  const Weights weight(value_of(best_key), greedy ? 1.f : temperature);

  // Visits the thread's tokens that lie at or above a key: f(logit, index).  A thread whose largest logit is below has none.
  const auto visit = [&](uint32_t least, auto f) {
    if (own_top < least) return;
    for (int i = tid; i < count; i += THREADS) {
      const Piece<T> p(held[i]);
#pragma unroll
      for (int e = 0; e < E; ++e) f(p.v[e], (from + i) * E - skew + e);
    }
  };
  // A token as one number, in falling order of which the prefixes are cut; all of them are different.
  const auto rank_of = [](float l, int token) { return ((unsigned long long)key_of(l) << 32) | (0xffffffffu - (uint32_t)token); };
  const auto logit_of = [](unsigned long long number) { return value_of((uint32_t)(number >> 32)); };

  // Who looks for a cut: the cluster, among all tokens, or the first block, among those of its list.
  const auto all_tokens = [&](unsigned long long least, auto f) {
    const float lowest = value_of((uint32_t)(least >> 32));
    visit((uint32_t)(least >> 32), [&](float l, int token) {
      if (!(l >= lowest)) return;
      const unsigned long long number = rank_of(l, token);
      if (number >= least) f(number);
    });
  };
  const auto listed_tokens = [&](unsigned long long least, auto f) {
    for (int i = tid; i < (int)sh.listed; i += THREADS)
      if (sh.list[i] >= least) f(sh.list[i]);
  };

  const auto clear_bins = [&] {
    for (int i = tid; i < BINS; i += THREADS) sh.count[i] = sh.low[i] = sh.high[i] = 0u;
    __syncthreads();
  };
  const auto put = [&](int bin, float l, bool masses, int k) {
    atomicAdd(&sh.count[bin], 1u);
    if (masses) {
      const uint32_t w = weight.mass(l, k);
      if (w != 0u) atomicAdd(&sh.low[bin], w & 0xffffu);
      if (w >> 16 != 0u) atomicAdd(&sh.high[bin], w >> 16);
    }
  };
  // Where the sum over the bins of `n` blocks, from the first bin on, reaches `target`: the n-th token, or that mass.  Returns
  // the sum of all bins; `target` of 0 stands for a share of it.  `k`: of the one bin that has been divided, or below 0.
  const auto cross = [&](auto wide, bool masses, double share, unsigned long long& target, int k) {
    constexpr bool WIDE = decltype(wide)::value;
    const int n = WIDE ? blocks : 1, me = WIDE ? rank : 0;
    const auto sync = [&] {
      if (WIDE) cluster.sync();
      else __syncthreads();
    };
    sync();  // every block's bins are complete
    const int slice = BINS / n;
    constexpr int PER = BINS / THREADS;
    const int own = max(1, PER / n);  // bins of one thread
    unsigned long long mine[PER], upto = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      mine[j] = 0;
      const int bin = me * slice + tid * own + j;
      if (j < own && tid * own + j < slice) {
#pragma unroll 2
        for (int r = 0; r < n; ++r) {  // several blocks' loads under way together
          if (masses) mine[j] += WIDE ? *peer(&sh.low[bin], r) + ((unsigned long long)*peer(&sh.high[bin], r) << 16)
                                      : sh.low[bin] + ((unsigned long long)sh.high[bin] << 16);
          else mine[j] += WIDE ? *peer(&sh.count[bin], r) : sh.count[bin];
        }
        if (masses) mine[j] <<= 13 - (k < 0 ? bin_power(bin) : k);
      }
      upto += mine[j];
    }
    const unsigned long long of_thread = upto;
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    unsigned long long sum = 0, base = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) upto += sh.scan[w];
      sum += sh.scan[w];
    }
    if (WIDE) {
      if (tid < n) *peer(&sh.slice[me], tid) = sum;
      cluster.sync();
      sum = 0;
      for (int r = 0; r < n; ++r) {
        if (r < me) base += sh.slice[r];
        sum += sh.slice[r];
      }
    }
    if (target == 0) target = (unsigned long long)ceil(fmax(share * (double)sum, 1.0));
    unsigned long long before = base + upto - of_thread;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j < own && before < target && target <= before + mine[j]) {
        Found found{me * slice + tid * own + j, 0u, before};
        for (int r = 0; r < n; ++r) found.count += WIDE ? *peer(&sh.count[found.bin], r) : sh.count[found.bin];
        for (int r = 0; r < n; ++r) *(WIDE ? peer(&sh.found, r) : &sh.found) = found;
      }
      before += mine[j];
    }
    sync();
    return sum;
  };

  // Adds tokens to the first block's list: each block collects its own, and asks for room once.  Returns how many they are.
  unsigned long long* const staging = reinterpret_cast<unsigned long long*>(sh.count);
  const auto gather = [&](const auto& each) {
    if (tid == 0) sh.staged = 0u;
    __syncthreads();
    each([&](unsigned long long number) {
      const uint32_t at = atomicAdd(&sh.staged, 1u);
      if (at < STAGED) staging[at] = number;
    });
    __syncthreads();
    const uint32_t mine = sh.staged;
    if (tid == 0) sh.room = atomicAdd(peer(&sh.listed, 0), mine);
    __syncthreads();
    for (uint32_t i = tid; i < min(mine, (uint32_t)STAGED); i += THREADS)
      if (sh.room + i < MEDIUM) *peer(&sh.list[sh.room + i], 0) = staging[i];
    return mine;
  };
  const auto smaller = [](unsigned long long x, unsigned long long y) { return x < y ? x : y; };
  using Cluster = std::integral_constant<bool, true>;
  using Block = std::integral_constant<bool, false>;

  // Tokens of one bin: those of a bin of the first histogram, or, once that has been divided, those between two bounds.
  struct Bin {
    int first;
    bool divided;
    unsigned long long low, high;
  };
  const auto in_bin = [&](const Bin& bin, unsigned long long number) {
    return bin.divided ? number <= bin.high : first_bin(weight, logit_of(number)) == bin.first;
  };
  // A histogram over the bin's tokens, by their numbers' bits; `bin` becomes the one of its 2048 parts that holds the target.
  const auto divide = [&](auto wide, const auto& tokens, Bin& bin, Found& found, bool masses, unsigned long long target) {
    constexpr bool WIDE = decltype(wide)::value;
    if (!bin.divided) {
      unsigned long long least = ~0ull, most = 0ull;
      tokens(bin.low, [&](unsigned long long number) {
        if (!in_bin(bin, number)) return;
        least = min(least, number);
        most = max(most, number);
      });
      least = block_reduce(least, sh.scan, smaller);
      most = block_reduce(most, sh.scan, better);
      if (WIDE) {
        if (tid < blocks) {
          *peer(&sh.ends[0][rank], tid) = least;
          *peer(&sh.ends[1][rank], tid) = most;
        }
        cluster.sync();
        for (int r = 0; r < blocks; ++r) {
          least = min(least, sh.ends[0][r]);
          most = max(most, sh.ends[1][r]);
        }
      }
      bin.divided = true;
      bin.low = least;
      bin.high = most;
    }
    const int shift = max(0, 64 - __clzll((long long)(bin.high - bin.low)) - 11);  // 2^11 bins
    clear_bins();
    tokens(bin.low, [&](unsigned long long number) {
      if (in_bin(bin, number)) put((int)((bin.high - number) >> shift), logit_of(number), masses, bin_power(bin.first));
    });
    unsigned long long left = target - found.before;
    cross(wide, masses, 0.0, left, bin_power(bin.first));
    const unsigned long long before = found.before + sh.found.before;
    found = sh.found;
    found.before = before;
    bin.high -= (unsigned long long)found.bin << shift;
    bin.low = max(bin.low, bin.high - ((1ull << shift) - 1));
  };

  // The lowest token of the shortest prefix of those at or above `cut` that holds `target` tokens, or that mass, or (target 0)
  // `share` of their mass; `cut` if there are not so many.  First among the listed ones, by the first block alone:
  const auto shorten_list = [&](unsigned long long cut, bool masses, double share, unsigned long long target) {
    clear_bins();
    listed_tokens(cut, [&](unsigned long long number) {
      const int bin = first_bin(weight, logit_of(number));
      put(bin, logit_of(number), masses, bin_power(bin));
    });
    if (cross(Block(), masses, share, target, -1) < target) return cut;
    Found found = sh.found;
    Bin bin{found.bin, false, cut, ~0ull};
    while (found.count > LIST) divide(Block(), listed_tokens, bin, found, masses, target);
    // rank the bin's tokens against one another
    listed_tokens(bin.low, [&](unsigned long long number) {
      if (!in_bin(bin, number)) return;
      const uint32_t at = atomicAdd(&sh.bin_listed, 1u);
      sh.bin_list[at] = number;
      sh.bin_mass[at] = masses ? weight.mass(logit_of(number), bin_power(bin.first)) : 1u;
    });
    __syncthreads();
    constexpr int PARTS = THREADS / LIST;
    const int mine = tid / PARTS;
    const unsigned long long me = mine < (int)found.count ? sh.bin_list[mine] : ~0ull;
    unsigned long long ahead = 0;
    for (int j = tid % PARTS; j < (int)found.count; j += PARTS)
      if (sh.bin_list[j] > me) ahead += sh.bin_mass[j];
    for (int o = PARTS / 2; o > 0; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    if (masses) ahead <<= 13 - bin_power(bin.first);
    const unsigned long long last = block_reduce(found.before + ahead < target ? me : ~0ull, sh.scan, smaller);
    if (tid == 0) sh.bin_listed = 0u;
    __syncthreads();
    return last;
  };
  // then among all: the cluster finds the bin, and sends its tokens to the first block.
  const auto shorten_row = [&](unsigned long long cut, bool masses, double share, unsigned long long target) {
    if (tid == 0) sh.listed = 0u;
    clear_bins();
    all_tokens(cut, [&](unsigned long long number) {
      const int bin = first_bin(weight, logit_of(number));
      put(bin, logit_of(number), masses, bin_power(bin));
    });
    if (cross(Cluster(), masses, share, target, -1) < target) return cut;
    Found found = sh.found;
    Bin bin{found.bin, false, cut, ~0ull};
    while (found.count > MEDIUM) divide(Cluster(), all_tokens, bin, found, masses, target);
    gather([&](const auto& f) {
      all_tokens(bin.low, [&](unsigned long long number) {
        if (in_bin(bin, number)) f(number);
      });
    });
    cluster.sync();
    if (rank == 0) {
      const unsigned long long last = shorten_list(0ull, masses, 0.0, target - found.before);
      if (tid < blocks) *peer(&sh.cut, tid) = last;
    }
    cluster.sync();
    return sh.cut;
  };

  Sums total;
  // ---- a short prefix: the tokens that reach the threshold, ranked by the first block
  threshold = max(threshold, 1u);
  {
    const float least = value_of(threshold);
    uint32_t sent = 0;
    unsigned long long sent_mass = 0;
    const auto send = [&](float l, int token) {
      if (!(l >= least && l > -INFINITY)) return;
      const uint32_t at = atomicAdd(peer(&sh.listed, 0), 1u);
      const unsigned long long mass = weight.mass(l);
      if (at < SHORT) {
        *peer(&sh.list[at], 0) = rank_of(l, token);
        *peer(&sh.list_mass[at], 0) = mass;
      }
      ++sent;
      sent_mass += mass;
    };
    for (int i = tid; i < count; i += THREADS) {
      const Piece<T> p(held[i]);
      float most = -INFINITY;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        total.add(weight.single ? pair(weight(p.v[e]), weight(p.v[e + 1])) : weight(pair(p.v[e], p.v[e + 1])));
        most = fmaxf(most, fmaxf(p.v[e], p.v[e + 1]));
      }
      if (!(most >= least && most > -INFINITY)) continue;
      const T* const held_tokens = reinterpret_cast<const T*>(held + i);
      for (int e = 0; e < E; ++e) send(Piece<T>::one(held_tokens[e]), (from + i) * E - skew + e);
    }
    double of_warp = total.value();
    sent = __reduce_add_sync(0xffffffffu, sent);
    for (int o = 16; o > 0; o >>= 1) {
      of_warp += __shfl_xor_sync(0xffffffffu, of_warp, o);
      sent_mass += __shfl_xor_sync(0xffffffffu, sent_mass, o);
    }
    if (lane == 0) {
      sh.reduce64[warp] = of_warp;
      sh.scan[warp] = sent_mass;
      sh.reduce32[warp] = sent;
    }
    __syncthreads();
    if (warp == 0) {
      of_warp = lane < WARPS ? sh.reduce64[lane] : 0.0;
      sent_mass = lane < WARPS ? sh.scan[lane] : 0ull;
      sent = __reduce_add_sync(0xffffffffu, lane < WARPS ? sh.reduce32[lane] : 0u);
      for (int o = WARPS / 2; o > 0; o >>= 1) {
        of_warp += __shfl_xor_sync(0xffffffffu, of_warp, o);
        sent_mass += __shfl_xor_sync(0xffffffffu, sent_mass, o);
      }
      of_warp = __shfl_sync(0xffffffffu, of_warp, 0);
      sent_mass = __shfl_sync(0xffffffffu, sent_mass, 0);
      if (lane < blocks) {
        *peer(&sh.totals[rank], lane) = of_warp;
        *peer(&sh.masses[rank], lane) = sent_mass;
        *peer(&sh.counts[rank], lane) = sent;
      }
    }
    cluster.sync();
    double whole = 0.0;
    unsigned long long held_mass = 0;
    uint32_t n = 0;
    for (int r = 0; r < blocks; ++r) {
      whole += sh.totals[r];
      held_mass += sh.masses[r];
      n += sh.counts[r];
    }
    unsigned long long limit = (unsigned long long)ceil(fmax((double)top_p * whole * MASS, 1.0));
    const bool holds = greedy || (by_count ? n >= (uint32_t)top_k : by_mass ? held_mass >= limit : min_p > 0.f && weight(least) < min_p);
    if (n <= SHORT && holds) {
      if (rank != 0) return;
      // `parts` neighbouring threads share a token
      int parts = 1;
      while (parts < 32 && (int)n * parts * 2 <= THREADS) parts *= 2;
      const int mine = tid / parts;
      const bool on = mine < (int)n;
      const unsigned long long me = on ? sh.list[mine] : 0ull;
      const unsigned long long my_mass = on ? sh.list_mass[mine] : 0ull;
      const int token = (int)(0xffffffffu - (uint32_t)me);
      const float luck = on && !greedy ? noise[token] : 1.f;
      uint32_t ahead = 0;
      unsigned long long mass_ahead = 0;
      if (on) {
        for (int j = tid % parts; j < (int)n; j += parts) {
          if (sh.list[j] > me) {
            ++ahead;
            mass_ahead += sh.list_mass[j];
          }
        }
      }
      for (int o = parts / 2; o > 0; o >>= 1) {
        ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        mass_ahead += __shfl_xor_sync(0xffffffffu, mass_ahead, o);
      }
      bool stays = on && (!by_count || ahead < (uint32_t)top_k);
      if (by_mass) {
        if (by_count) {
          const unsigned long long left =
              block_reduce(stays && tid % parts == 0 ? my_mass : 0ull, sh.scan, [](unsigned long long x, unsigned long long y) { return x + y; });
          limit = (unsigned long long)ceil(fmax((double)top_p * (double)left, 1.0));
        }
        stays = stays && mass_ahead < limit;
      }
      const float l = value_of((uint32_t)(me >> 32)), w = weight(l);
      stays = stays && (greedy ? ahead == 0 : w >= min_p || l == weight.best);
      const float score = stays ? fmaxf(__fdividef(w, luck), -0.5f) : -1.f;
      const unsigned long long first =
          block_reduce(((unsigned long long)key_of(score) << 32) | (0xffffffffu - (uint32_t)token), sh.scan, better);
      if (tid == 0) {
        const int drawn = (int)(0xffffffffu - (uint32_t)first);
        a.token[row] = drawn;
        a.logprob[row] = (weight.exponent(Piece<T>::one(logits[drawn])) - __log2f((float)whole)) * LN2;
      }
      return;
    }
  }

  // ---- a longer one, or all tokens
  double whole = 0.0;
  for (int r = 0; r < blocks; ++r) whole += sh.totals[r];
  const unsigned long long limit = (unsigned long long)ceil(fmax((double)top_p * whole * MASS, 1.0));
  float best_score = -1.f;
  uint32_t winner = 0xffffffffu;
  const auto enter = [&](float l, float luck, uint32_t token) {  // a token into the race
    const float w = weight(l);
    if (l != weight.best && (greedy || !(w >= min_p))) return;
    const float score = greedy ? 1.f : fmaxf(__fdividef(w, luck), -0.5f);
    if (score > best_score || (score == best_score && token < winner)) {
      best_score = score;
      winner = token;
    }
  };
  const auto best_of_block = [&] {  // (score, lowest index) as one ordered number
    return block_reduce(((unsigned long long)key_of(best_score) << 32) | (0xffffffffu - winner), sh.scan, better);
  };
  const auto finish = [&](unsigned long long first) {
    if (tid != 0) return;
    const int token = (int)(0xffffffffu - (uint32_t)first);
    a.token[row] = token;
    a.logprob[row] = (weight.exponent(Piece<T>::one(logits[token])) - __log2f((float)whole)) * LN2;
  };
  unsigned long long cut = 1ull << 32;  // all but -inf
  if (by_count || by_mass) {
    if (tid == 0) sh.listed = 0u;
    cluster.sync();
    unsigned long long sent_mass = 0;
    const uint32_t sent = gather([&](const auto& f) {
      all_tokens((unsigned long long)max(lower, 1u) << 32, [&](unsigned long long number) {
        f(number);
        sent_mass += weight.mass(logit_of(number));
      });
    });
    sent_mass = block_reduce(sent_mass, sh.scan, [](unsigned long long x, unsigned long long y) { return x + y; });
    if (tid < blocks) {
      *peer(&sh.masses[rank], tid) = sent_mass;
      *peer(&sh.counts[rank], tid) = sent;
    }
    cluster.sync();
    unsigned long long held_mass = 0;
    uint32_t n = 0;
    for (int r = 0; r < blocks; ++r) {
      held_mass += sh.masses[r];
      n += sh.counts[r];
    }
    if (n <= MEDIUM && (by_count ? n >= (uint32_t)top_k : held_mass >= limit)) {
      if (rank != 0) return;
      if (by_count) cut = shorten_list(cut, false, 0.0, top_k);
      if (by_mass) cut = shorten_list(cut, true, top_p, by_count ? 0 : limit);
      listed_tokens(cut, [&](unsigned long long number) {
        const uint32_t token = 0xffffffffu - (uint32_t)number;
        enter(logit_of(number), noise[token], token);
      });
      finish(best_of_block());
      return;
    }
    if (by_count) cut = shorten_row(cut, false, 0.0, top_k);
    if (by_mass) cut = shorten_row(cut, true, top_p, by_count ? 0 : limit);
  }
  if (own_top >= (uint32_t)(cut >> 32)) {
    // pieces with a token that stays; the random numbers of several are under way together
    constexpr int DEPTH = E == 4 ? 4 : 2;
    const bool together = (reinterpret_cast<uintptr_t>(noise - skew) % 16) == 0;
    // number >= cut, without working the number out; -inf never stays (places in front of the row hold it, with indices below 0)
    const float lowest = value_of((uint32_t)(cut >> 32));
    const int last = lowest == -INFINITY ? INT_MIN : (int)min(0xffffffffu - (uint32_t)cut, 0x7fffffffu);
    const auto stays = [&](float l, int token) { return l > lowest || (l == lowest && token <= last); };
    for (int i0 = tid; i0 < count; i0 += DEPTH * THREADS) {
      float luck[DEPTH][E];
      bool any[DEPTH];
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        const int i = i0 + j * THREADS, first = (from + i) * E - skew;
        any[j] = false;
        if (i < count) {
          const Piece<T> p(held[i]);
#pragma unroll
          for (int e = 0; e < E; ++e) any[j] |= stays(p.v[e], first + e);
        }
        if (!any[j]) continue;
        if (together && inside(i)) {
#pragma unroll
          for (int x = 0; x < E / 4; ++x) {
            const float4 v = *(reinterpret_cast<const float4*>(noise + first) + x);
            luck[j][4 * x] = v.x, luck[j][4 * x + 1] = v.y, luck[j][4 * x + 2] = v.z, luck[j][4 * x + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) luck[j][e] = first + e >= 0 && first + e < a.V ? noise[first + e] : 1.f;
        }
      }
#pragma unroll
      for (int j = 0; j < DEPTH; ++j) {
        if (!any[j]) continue;
        const int i = i0 + j * THREADS, first = (from + i) * E - skew;
        const Piece<T> p(held[i]);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (stays(p.v[e], first + e)) enter(p.v[e], luck[j][e], (uint32_t)(first + e));
      }
    }
  }
  const unsigned long long first = best_of_block();
  if (tid == 0) *peer(&sh.slice[rank], 0) = first;
  cluster.sync();
  if (rank == 0) {
    unsigned long long most = 0;
    for (int r = 0; r < blocks; ++r) most = better(most, sh.slice[r]);
    finish(most);
  }
}

// Bytes of a row that let two blocks share an SM's 228 KB, of which each block takes another 1 KB.
constexpr long long STRETCH = (228 * 1024 / 2 - 1024 - (long long)(sizeof(Shared) + 15) / 16 * 16) / 16 * 16;
// Bytes that a block holds of a row that `blocks` share, at the worst alignment.
static long long stretch(const Args& a, int blocks) {
  const long long size = a.wide ? 4 : 2, pieces = (a.V * size + 2 * (16 - size)) / 16;
  return (pieces + blocks - 1) / blocks * 16;
}

// Blocks per row: as many as let two of them share an SM (512 rows of 36800 in bf16 57.8 us; with one block of 74 KB per row
// and SM 65.3), and more while all of them run at once and have some tokens for each thread.
static int blocks_per_row(const Args& a, int sms) {
  int blocks = 1;
  while (blocks < MOST_BLOCKS && stretch(a, blocks) > STRETCH) blocks *= 2;
  while (blocks < MOST_BLOCKS && (long long)a.B * blocks <= sms && a.V > blocks * 4096) blocks *= 2;
  return blocks;
}

template <typename T>
static cudaError_t launch_as(const Args& a, int blocks, cudaStream_t stream) {
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)stretch(a, blocks);
  // dynamic shared memory beyond 48 KB is opted into once per device, for the longest stretch of a block
  static unsigned long long opted = 0;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(__atomic_load_n(&opted, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(sizeof(Shared) + 64 + std::max<long long>(STRETCH, kMaxVocabulary / MOST_BLOCKS * sizeof(T))));
    if (err != cudaSuccess) return err;
    __atomic_fetch_or(&opted, bit, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(a.B * blocks));
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = blocks;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = a.streamed ? 2 : 1;
  return cudaLaunchKernelEx(&config, sample_kernel<T>, a);
}

// Rows of which nothing is cut, at an ordinary temperature, are streamed by persistent blocks where clusters of two blocks or
// more would need a second wave: 64 rows of 128256 in fp32 21.1 us against 23.1, 256 rows 47 against 81, in bf16 128 rows 27.3
// against 30.2.  With one wave (32 rows in fp32 15.6 against 11.6 us) or one block per row (512 rows of 32000 in bf16 32.0 against
// 29.5, 1024 of 16384 in fp32 42 against 38.6) clusters are faster.  Where a block fills an SM a wave is half as many: 24 rows of
// 262144 in fp32 23.0 us streamed against 25.5, 37 rows 26.6 against 40.4.
// Where temperature or filters are per row, only the device knows which rows those are: both kernels are launched, and each
// leaves the other's rows alone; the second begins as SMs get free (256 rows of 128256 in fp32: 54.7 us, 58 after the first's end).
// That pays from four blocks per row and two waves on: those 256 rows 54.7 us against 83, 96 rows 27.9 against 34.1, 192 in bf16
// 37.5 against 44.3; 48 of 262144 in fp32 32.8 against 53.6; 64 rows in fp32 24.1 against 23.1, 128 in bf16 31.1 against 30.2.  Batches that turn out to be cut lose the
// time of a launch (256 rows of top-k 1000: 165 -> 170 us; 70 of 262144 in fp32 with top-p 0.9: 63.7 -> 69.8).
static bool whole_stream(const Args& a) {
  if (a.temperature.rows != nullptr) return false;
  if (a.temperature.same <= 0.f) return true;
  return ordinary(a.temperature.same) && a.top_k.rows == nullptr && a.top_p.rows == nullptr && a.min_p.rows == nullptr &&
         cuts_nothing(a.top_k.same, a.top_p.same, a.min_p.same, a.V);
}

bool streams(const Args& a, int sms) {
  const int blocks = blocks_per_row(a, sms);
  const long long wave = (stretch(a, blocks) <= STRETCH ? 2ll : 1ll) * sms;  // blocks that run at once
  if (blocks == 1 || (long long)a.B * blocks <= wave) return false;
  // what the streaming kernel counts in 32 bits, and the rows of one block that it can put off
  if (whole_stream(a)) return (long long)a.B * (a.V / 4 + 2) < (1ll << 31) && a.B / sms < 1000;
  if (blocks < 4 || (long long)a.B * blocks <= 2 * wave || a.B > kMostListed) return false;
  return (a.temperature.rows != nullptr || ordinary(a.temperature.same)) &&
         cuts_nothing(a.top_k.rows != nullptr ? 0 : a.top_k.same, a.top_p.rows != nullptr ? 1.f : a.top_p.same,
                      a.min_p.rows != nullptr ? 0.f : a.min_p.same, a.V);
}

cudaError_t launch(const Args& args, int sms, cudaStream_t stream) {
  Args a = args;
  a.streamed = streams(a, sms);
  if (a.streamed) {
    const cudaError_t err = launch_stream(a, whole_stream(a), sms, stream);
    if (err != cudaSuccess || whole_stream(a)) return err;
  }
  const int blocks = blocks_per_row(a, sms);
  return a.wide ? launch_as<float>(a, blocks, stream) : launch_as<__nv_bfloat16>(a, blocks, stream);
}

}  // namespace sampling
}  // namespace ht
