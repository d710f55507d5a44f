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
// rows, the latency of the steps.  A row belongs to a cluster of blocks.  Each block holds its stretch of
// the row in shared memory, so the row is read from memory once, and the cluster exchanges a few numbers
// per step through distributed shared memory.
//
// * A cut is found without sorting: one histogram of all tokens over 2048 bins of falling logit (a bin per
//   1/256 of an octave of 1 + distance from the best: narrow where the mass is), whose bins hold
//   counts for top_k and masses for top_p, then the one bin that holds the boundary is resolved: its tokens
//   are gathered and ranked against one another, or, if there are many, divided further by their bits.
// * Masses are integers, round(w 2^31), split into halves of 16 bits that 32-bit shared-memory atomics add
//   without overflow.  Integer sums do not depend on their order, so neither does the result.
// * The total for the log-probability is summed so that its order does not show either (Sum).
#include <cooperative_groups.h>

#include "generation.cuh"

namespace cg = cooperative_groups;

namespace ht {
namespace sampling {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 2048;
constexpr int LIST = 1024;      // tokens of one bin that are ranked directly
constexpr int MOST_BLOCKS = 8;  // of a cluster
constexpr float LN2 = 0.6931471805599453f;

// Unsigned keys in the order of the floats; -inf has the lowest one.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(l + 0.f);  // -0 + 0 = +0: equal logits have equal keys
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return key == 0u ? -INFINITY : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// w = 2^((l - best) log2(e) / T); the quotient is carried in two floats, since its rounding error times the distance
// would show in the weights of unlikely tokens.
struct Weights {
  float best, hi, lo, least;
  bool single;  // only tokens equal to the best weigh anything (best = +inf, or 1 / T beyond fp32)
  __device__ Weights(float best_, float temperature) : best(best_) {
    const double rate = 1.4426950408889634 / fmin((double)temperature, 1e30);
    hi = (float)rate;
    single = best == INFINITY || hi == INFINITY;
    lo = single ? 0.f : (float)(rate - (double)hi);
    least = single ? 0.f : -2048.f / hi;  // further away the weight is zero whatever the correction says
  }
  __device__ __forceinline__ float exponent(float l) const {
    if (single) return l == best ? 0.f : -INFINITY;
    const float d = l - best;
    return fmaf(d, hi, fmaxf(d, least) * lo);
  }
  __device__ __forceinline__ float operator()(float l) const { return fast_exp2(exponent(l)); }
  __device__ __forceinline__ uint32_t fixed(float l) const { return (uint32_t)__float2uint_rn((*this)(l)*2147483648.f); }
};

// A sum of weights that comes out the same in every order (and so for every alignment of the row): multiples of 2^-16,
// which a thread's few hundred terms add without rounding, and what they leave of each weight (at most 2^-17), whose
// roundings lie far below the fp32 result.
struct Sum {
  float coarse = 0.f, fine = 0.f;
  __device__ __forceinline__ void add(float w) {
    const float near = __fadd_rn(__fadd_rn(w, 128.f), -128.f);
    coarse += near;
    fine += w - near;
  }
  __device__ __forceinline__ double value() const { return (double)coarse + (double)fine; }
};

struct Found {  // where a running sum over the bins crosses its target
  int bin;
  uint32_t count;            // tokens of the bin
  unsigned long long before;  // sum of the bins in front of it
};

struct Shared {
  uint32_t count[BINS], low[BINS], high[BINS];  // masses: 2^16 high + low
  unsigned long long list[LIST];
  uint32_t list_mass[LIST];
  uint32_t listed;
  unsigned long long scan[WARPS];
  uint32_t reduce32[WARPS];
  unsigned long long slice[MOST_BLOCKS];                      // per block of the cluster
  uint32_t keys[2][MOST_BLOCKS], ties[MOST_BLOCKS];           // likewise
  double totals[MOST_BLOCKS], reduce64[WARPS];                // likewise
  Found found;
  unsigned long long cut;
};

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* scratch, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
  __syncthreads();
  v = scratch[threadIdx.x % WARPS];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// 16 bytes of the row as floats.
template <typename T>
struct Piece {
  static constexpr int E = 16 / sizeof(T);
  float v[E];
  static __device__ __forceinline__ float one(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return __bfloat162float(x);
  }
  __device__ __forceinline__ explicit Piece(uint4 raw) {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        v[j] = __uint_as_float(u[j]);
      } else {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
      }
    }
  }
};

// A bin per 1/256 of an octave of 1 + x / 2: bins of 1/128 up to a distance of 2, of 1/64 up to 6, and so on; all tokens
// beyond 510 share the last bin.  Monotone in l, as every step of its computation is.
__device__ __forceinline__ int first_bin(const Weights& weight, float l) {
  const float away = fmaf(weight.exponent(l), -0.5f * LN2, 1.f);
  return min((int)(min(__float_as_uint(away), 0x43800000u) >> 15) - (0x3f800000 >> 15), BINS - 1);
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Args a) {
  constexpr int E = Piece<T>::E;
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& sh = *reinterpret_cast<Shared*>(smem);
  uint4* const held = reinterpret_cast<uint4*>(smem + (sizeof(Shared) + 15) / 16 * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / blocks, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const auto peer = [&](auto* p, int r) { return cluster.map_shared_rank(p, r); };

  // ---- this block's stretch of the row, as aligned pieces of 16 bytes; places outside the row hold -inf
  const T* const logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int skew = (int)((reinterpret_cast<uintptr_t>(logits) % 16) / sizeof(T));
  const uint4* const aligned = reinterpret_cast<const uint4*>(logits - skew);
  const int pieces = (skew + a.V + E - 1) / E, each = (pieces + blocks - 1) / blocks;
  const int from = min(rank * each, pieces), count = min(each, pieces - from);
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
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
  const auto inside = [&](int i) {  // whether all of the piece belongs to the row
    const int first = (from + i) * E - skew;
    return first >= 0 && first + E <= a.V;
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
        if (!inside(i)) {  // the row's ends
          uint32_t u[4] = {none, none, none, none};
          for (int e = 0; e < E; ++e) {
            const int token = (from + i) * E - skew + e;
            if (token < 0 || token >= a.V) continue;
            if constexpr (sizeof(T) == 4) u[e] = __float_as_uint(logits[token]);
            else u[e / 2] = (u[e / 2] & (e % 2 ? 0xffffu : 0xffff0000u)) | ((uint32_t)__bfloat16_as_ushort(logits[token]) << (16 * (e % 2)));
          }
          raw[j] = make_uint4(u[0], u[1], u[2], u[3]);
        }
        keep_piece(i, raw[j]);
      }
    }
  }
  const auto larger = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
  const uint32_t own_top = key_of(top);
  uint32_t best_key = block_reduce(own_top, sh.reduce32, larger);
  if (tid < blocks) *peer(&sh.keys[0][rank], tid) = best_key;
  cluster.sync();
  for (int r = 0; r < blocks; ++r) best_key = max(best_key, sh.keys[0][r]);
  if (best_key == 0u) {  // the same for every block of the cluster
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      a.logprob[row] = -INFINITY;
    }
    return;
  }

  const float temperature = a.temperature[row];
  const bool greedy = !(temperature > 0.f);
  const Weights weight(value_of(best_key), greedy ? 1.f : temperature);
  const int top_k = a.top_k[row];
  const float top_p = a.top_p[row];
  const bool by_count = !greedy && top_k > 0 && top_k < a.V, by_mass = !greedy && !(top_p >= 1.f);

  // Visits the thread's tokens that lie at or above a key: f(logit, index).  A thread whose largest logit is below has none.
  const auto visit = [&](uint32_t least, auto f) {
    if (own_top < least) return;
    for (int i = tid; i < count; i += THREADS) {
      const Piece<T> p(held[i]);
#pragma unroll
      for (int e = 0; e < E; ++e) f(p.v[e], (from + i) * E - skew + e);
    }
  };
  // A token as one number, in falling order of which the prefixes are cut.
  const auto rank_of = [](float l, int token) { return ((unsigned long long)key_of(l) << 32) | (0xffffffffu - (uint32_t)token); };

  unsigned long long cut = 1ull << 32;  // tokens at or above it stay: at first all but -inf

  const auto clear_bins = [&] {
    for (int i = tid; i < BINS; i += THREADS) sh.count[i] = sh.low[i] = sh.high[i] = 0u;
    if (tid == 0) sh.listed = 0u;
    __syncthreads();
  };
  const auto put = [&](int bin, float l, bool masses) {
    atomicAdd(&sh.count[bin], 1u);
    if (masses) {
      const uint32_t w = weight.fixed(l);
      if (w != 0u) atomicAdd(&sh.low[bin], w & 0xffffu);
      if (w >> 16 != 0u) atomicAdd(&sh.high[bin], w >> 16);
    }
  };
  // The sum over all bins of all blocks, and where the sum from the first bin on reaches `target` (of a share of the sum).
  const auto cross = [&](bool masses, double share, unsigned long long target, unsigned long long& sum) {
    cluster.sync();  // every block's bins are complete
    const int slice = BINS / blocks;
    constexpr int PER = BINS / THREADS;
    const int own = min(PER, slice * PER / BINS + (slice * PER % BINS ? 1 : 0));  // bins of one thread
    unsigned long long mine[PER], upto = 0;
    uint32_t counts[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      mine[j] = 0;
      counts[j] = 0;
      const int bin = rank * slice + tid * own + j;
      if (j < own && tid * own + j < slice) {
        for (int r = 0; r < blocks; ++r) {
          const uint32_t c = *peer(&sh.count[bin], r);
          counts[j] += c;
          mine[j] += masses ? *peer(&sh.low[bin], r) + ((unsigned long long)*peer(&sh.high[bin], r) << 16) : c;
        }
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
    unsigned long long total = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) upto += sh.scan[w];
      total += sh.scan[w];
    }
    if (tid < blocks) *peer(&sh.slice[rank], tid) = total;
    cluster.sync();
    sum = 0;
    unsigned long long base = 0;
    for (int r = 0; r < blocks; ++r) {
      if (r < rank) base += sh.slice[r];
      sum += sh.slice[r];
    }
    if (masses && target == 0) target = max(1ull, (unsigned long long)ceil(share * (double)sum));
    unsigned long long before = base + upto - of_thread;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (j < own && before < target && target <= before + mine[j]) {
        const Found found{rank * slice + tid * own + j, counts[j], before};
        for (int r = 0; r < blocks; ++r) *peer(&sh.found, r) = found;
      }
      before += mine[j];
    }
    cluster.sync();
    return target;
  };

  // Cuts to the shortest prefix that holds `target` tokens, or `share` of the mass of what is left.
  const auto shorten = [&](bool masses, double share, unsigned long long target) {
    unsigned long long sum = 0;
    target = cross(masses, share, target, sum);
    if (sum < target) return;  // fewer tokens than top_k
    Found found = sh.found;
    uint32_t low_key = 0, high_key = 0;  // of the bin's tokens, once it has been divided
    bool divided = false;
    int bin = found.bin;
    unsigned long long before = found.before;
    const auto member = [&](float l, int token) {
      if (rank_of(l, token) < cut) return false;
      return divided ? key_of(l) >= low_key && key_of(l) <= high_key : first_bin(weight, l) == bin;
    };
    while (found.count > LIST && !(divided && low_key == high_key)) {
      if (!divided) {
        uint32_t least = 0xffffffffu, most = 0u;
        visit((uint32_t)(cut >> 32), [&](float l, int token) {
          if (member(l, token)) {
            least = min(least, key_of(l));
            most = max(most, key_of(l));
          }
        });
        least = block_reduce(least, sh.reduce32, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
        most = block_reduce(most, sh.reduce32, larger);
        if (tid < blocks) {
          *peer(&sh.keys[0][rank], tid) = least;
          *peer(&sh.keys[1][rank], tid) = most;
        }
        cluster.sync();
        low_key = 0xffffffffu;
        for (int r = 0; r < blocks; ++r) {
          low_key = min(low_key, sh.keys[0][r]);
          high_key = max(high_key, sh.keys[1][r]);
        }
        divided = true;
        continue;
      }
      int shift = 0;
      while ((high_key - low_key) >> shift >= BINS) ++shift;
      clear_bins();
      visit(low_key, [&](float l, int token) {
        if (member(l, token)) put((high_key - key_of(l)) >> shift, l, masses);
      });
      cross(masses, share, target - before, sum);
      found = sh.found;
      before += found.before;
      high_key -= (uint32_t)found.bin << shift;
      low_key = max(low_key, high_key - (uint32_t)((1ull << shift) - 1));
    }
    if (found.count <= LIST) {
      // The first block ranks the bin's tokens against one another.
      visit(divided ? low_key : (uint32_t)(cut >> 32), [&](float l, int token) {
        if (!member(l, token)) return;
        const uint32_t at = atomicAdd(peer(&sh.listed, 0), 1u);
        *peer(&sh.list[at], 0) = rank_of(l, token);
        *peer(&sh.list_mass[at], 0) = masses ? weight.fixed(l) : 1u;
      });
      cluster.sync();
      if (rank == 0) {
        unsigned long long last = ~0ull;
        for (int i = tid; i < (int)found.count; i += THREADS) {
          const unsigned long long mine = sh.list[i];
          unsigned long long ahead = before;
          for (int j = 0; j < (int)found.count; ++j)
            if (sh.list[j] > mine) ahead += sh.list_mass[j];
          if (ahead < target) last = min(last, mine);
        }
        last = block_reduce(last, sh.scan, [](unsigned long long x, unsigned long long y) { return x < y ? x : y; });
        if (tid < blocks) *peer(&sh.cut, tid) = last;
      }
      cluster.sync();
      cut = sh.cut;
      return;
    }
    // Many equal logits: the first n of them, in the order of their index, stay.
    const unsigned long long w = masses ? weight.fixed(value_of(high_key)) : 1ull;
    unsigned long long n = (target - before + w - 1) / w;
    uint32_t equal = 0;
    visit(high_key, [&](float l, int token) { equal += key_of(l) == high_key && rank_of(l, token) >= cut; });
    const uint32_t of_block = block_reduce(equal, sh.reduce32, [](uint32_t x, uint32_t y) { return x + y; });
    if (tid < blocks) *peer(&sh.ties[rank], tid) = of_block;
    cluster.sync();
    for (int r = 0; r < rank; ++r) n -= min(n, (unsigned long long)sh.ties[r]);
    if (n >= 1 && n <= of_block) {  // the last one is in this block: count on in the order of the index
      uint32_t seen = 0;
      for (int i0 = 0; i0 < count; i0 += THREADS) {
        uint32_t here = 0;
        const int i = i0 + tid;
        if (i < count) {
          const Piece<T> p(held[i]);
#pragma unroll
          for (int e = 0; e < E; ++e) here += key_of(p.v[e]) == high_key && rank_of(p.v[e], (from + i) * E - skew + e) >= cut;
        }
        uint32_t upto = here;
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t other = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += other;
        }
        __syncthreads();
        if (lane == 31) sh.reduce32[warp] = upto;
        __syncthreads();
        uint32_t all = 0;
        for (int x = 0; x < WARPS; ++x) {
          if (x < warp) upto += sh.reduce32[x];
          all += sh.reduce32[x];
        }
        uint32_t ahead = seen + upto - here;
        if (ahead < n && n <= ahead + here) {
          const Piece<T> p(held[i]);
          for (int e = 0; e < E; ++e) {
            const int token = (from + i) * E - skew + e;
            if (key_of(p.v[e]) == high_key && rank_of(p.v[e], token) >= cut && ++ahead == n)
              for (int r = 0; r < blocks; ++r) *peer(&sh.cut, r) = rank_of(p.v[e], token);
          }
        }
        seen += all;
      }
    }
    cluster.sync();
    cut = sh.cut;
  };

  Sum total;
  if (by_count || by_mass) {
    clear_bins();
    const bool masses = !by_count;
    visit(0u, [&](float l, int) {
      total.add(weight(l));
      if (l > -INFINITY) put(first_bin(weight, l), l, masses);
    });
    shorten(masses, top_p, by_count ? top_k : 0);
    if (by_count && by_mass) {
      clear_bins();
      visit((uint32_t)(cut >> 32), [&](float l, int token) {
        if (rank_of(l, token) >= cut) put(first_bin(weight, l), l, true);
      });
      shorten(true, top_p, 0);
    }
  }

  // ---- the race
  const float min_p = a.min_p[row];
  const float* const noise = a.noise + row * a.noise_stride;
  float best_score = -1.f;
  int winner = a.V;
  const auto run = [&](float l, float e, int token) {
    const float w = weight(l);
    // a NaN (from a random number that is none) loses to every score, but still names a token
    const float score = fmaxf(__fdividef(w, e), -0.5f);
    if (score > best_score && (w >= min_p || l == weight.best)) {
      best_score = score;
      winner = token;
    }
    return w;
  };
  if (greedy) {
    visit(0u, [&](float l, int token) {
      total.add(weight(l));
      if (l == weight.best && token < winner) winner = token, best_score = 1.f;
    });
  } else if (by_count || by_mass) {
    visit((uint32_t)(cut >> 32), [&](float l, int token) {
      if (rank_of(l, token) >= cut) run(l, noise[token], token);
    });
  } else if (min_p > 0.f) {
    visit(0u, [&](float l, int token) {
      const float w = weight(l);
      total.add(w);
      if (w >= min_p || l == weight.best) run(l, noise[token], token);
    });
  } else {
    // every token: whole pieces of the random numbers where the two rows are aligned to one another
    const bool together = (reinterpret_cast<uintptr_t>(noise - skew) % 16) == 0;
    for (int i = tid; i < count; i += THREADS) {
      const Piece<T> p(held[i]);
      const int first = (from + i) * E - skew;
      float e[E];
      if (together && inside(i)) {
#pragma unroll
        for (int j = 0; j < E / 4; ++j) {
          const float4 x = __ldcs(reinterpret_cast<const float4*>(noise + first) + j);
          e[4 * j] = x.x, e[4 * j + 1] = x.y, e[4 * j + 2] = x.z, e[4 * j + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = first + j >= 0 && first + j < a.V ? noise[first + j] : 1.f;
      }
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (p.v[j] > -INFINITY) total.add(run(p.v[j], e[j], first + j));
    }
  }

  // ---- over the block and the cluster
  const double of_block = block_reduce(total.value(), sh.reduce64, [](double x, double y) { return x + y; });
  const auto better = [](unsigned long long x, unsigned long long y) { return x > y ? x : y; };
  const unsigned long long first_of =
      block_reduce(((unsigned long long)key_of(best_score) << 32) | (0xffffffffu - (uint32_t)winner), sh.scan, better);
  if (tid == 0) {
    *peer(&sh.totals[rank], 0) = of_block;
    *peer(&sh.slice[rank], 0) = first_of;
  }
  cluster.sync();
  if (rank == 0 && tid == 0) {
    unsigned long long most = 0;
    double sum = 0.0;
    for (int r = 0; r < blocks; ++r) {
      most = better(most, sh.slice[r]);
      sum += sh.totals[r];
    }
    const int token = (int)(0xffffffffu - (uint32_t)most);
    const float l = Piece<T>::one(logits[token]);
    a.token[row] = token;
    a.logprob[row] = (weight.exponent(l) - __log2f((float)sum)) * LN2;
  }
}

template <typename T>
static cudaError_t launch_as(const Args& a, int blocks, cudaStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int pieces = (a.V + 2 * E - 2) / E, each = (pieces + blocks - 1) / blocks;
  const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)each * 16;
  // dynamic shared memory beyond 48 KB is opted into once per device, for the largest vocabulary
  static unsigned long long opted = 0;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(__atomic_load_n(&opted, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(sizeof(Shared) + 64 + (kMaxVocabulary / MOST_BLOCKS) * sizeof(T)));
    if (err != cudaSuccess) return err;
    __atomic_fetch_or(&opted, bit, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(a.B * blocks));
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = blocks;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, sample_kernel<T>, a);
}

cudaError_t launch(const Args& a, int sms, cudaStream_t stream) {
  // blocks per row: a block of 512 threads with at least a piece of 16 bytes for each, at most 8
  int blocks = 1;
  while (blocks < MOST_BLOCKS && a.V > blocks * 4096) blocks *= 2;
  return a.wide ? launch_as<float>(a, blocks, stream) : launch_as<__nv_bfloat16>(a, blocks, stream);
}

}  // namespace sampling
}  // namespace ht
