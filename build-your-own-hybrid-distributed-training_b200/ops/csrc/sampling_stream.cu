// Choosing the next token where nothing is cut: many rows of logits and random numbers, streamed once.
//
// With w_i = 2^(l_i log2(e) / T) the token with the largest w_i / e_i is taken, and its log-probability is
// log(w_i / sum w).  T <= 0 takes the first of the largest logits (and T = 1 for the log-probability).
//
// Bound: memory.  All rows form one line of 16-byte pieces, cut into equal stretches, one for a persistent block on every SM.
// Each warp copies its own pieces into a ring in shared memory, turns ahead and across the ends of rows, so
// that the loads never stop: 256 rows of 128256 in fp32 take 47 us (floor 40), against 81 us with a cluster per row, which
// has all loads of its row under way but none of the next one's.  (Two blocks of half the threads per SM finish up to a third
// apart: 48 us.)  A bf16 piece's random numbers are copied by neighbouring lanes, not by the lane that uses them, whose
// 16-byte reads 32 bytes apart would fetch every sector twice: 512 rows of bf16 79 against 93 us.
//
// A warp keeps one reference for its exponents, an integer that rises with the largest logit so far, and the
// best score so far.  At the end of a row, or of the block's part of it, the warps' (reference, sum, best token) are merged by
// one warp while the others go on; rows that cross blocks go through a workspace, where the block that arrives last
// merges the parts in their order, so that results do not depend on timing.  Rows whose logits leave the range in which one
// reference serves (beyond 1e5 in the exponent, or infinite) are put off and done by their block one after the other: a batch of
// nothing else takes 264 us for 256 rows of 128256 in fp32, and 71 for 160 of 50257 in bf16 (ordinary ones 51.5 and 32).
//
// Sums of weights are fp32: a thread adds at most some 256 of a row, whose roundings leave 5e-8 of the log-probability, as much
// as its own rounding.
#include "sampling.cuh"

namespace ht {
namespace sampling {

namespace {

constexpr int WIDTH = 1024, GROUPS = WIDTH / 32;  // threads and warps of a block
constexpr int MOST_ROWS = 1024;  // of one block
constexpr uint32_t NOBODY = 0xffffffffu;  // no token yet

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// What a warp or a block knows of a row.
struct alignas(16) Part {
  float reference, sum;  // of 2^(x - reference)
  uint32_t key, token;   // of the best score (greedy: logit)
};
__device__ __forceinline__ Part load(const Part* p) {  // of this block's shared memory, or written by a block before it arrived
  Part v;
  asm volatile("ld.relaxed.gpu.v4.b32 {%0, %1, %2, %3}, [%4];" : "=f"(v.reference), "=f"(v.sum), "=r"(v.key), "=r"(v.token) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned arrive(unsigned* counter) {  // publishes this thread's writes, and shows it those before it
  unsigned before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}

struct Small {
  Part parts[2][GROUPS];
  int rows[MOST_ROWS];  // left for the end: infinite or huge logits
  int count, counts[GROUPS];
  double sums[GROUPS];
  unsigned long long picks[GROUPS];
};

struct Listed {
  int row;
  float temperature;
};

template <bool GREEDY, typename T>
struct Ring {
  static constexpr int E = Piece<T>::E, PER = 8 / E;             // pieces of a thread in one turn: 8 tokens
  static constexpr int UNITS = PER + (GREEDY ? 0 : 2);           // 16 bytes of logits or random numbers
  static constexpr int STAGES = UNITS >= 2 ? 12 / UNITS : 8;     // 192 KB or, of greedy bf16, 128
  static constexpr int BYTES = STAGES * UNITS * WIDTH * 16;
};

// WHOLE: all rows are this kernel's, at one temperature, whose log2(e) / T is hi + lo.
template <bool GREEDY, bool WHOLE, typename T>
__global__ void __launch_bounds__(WIDTH, 1)
stream_kernel(const __grid_constant__ Args a, int pieces /* of a row's share of the line */, float hi, float lo) {
  using R = Ring<GREEDY, T>;
  constexpr int E = R::E, PER = R::PER, UNITS = R::UNITS, STAGES = R::STAGES, TURN = PER * WIDTH;
  extern __shared__ __align__(16) unsigned char smem[];
  // A stage of the ring: the pieces of all threads, then their random numbers, a warp's together.
  uint4* const ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;
  float* const lucks = reinterpret_cast<float*>(smem) + (PER * WIDTH * 4 + threadIdx.x / 32 * 32 * E);
  Small& sh = *reinterpret_cast<Small*>(smem + R::BYTES);
  Listed* const listed = reinterpret_cast<Listed*>(smem + R::BYTES + sizeof(Small));  // not if WHOLE
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;

  if constexpr (!WHOLE) asm volatile("griddepcontrol.launch_dependents;");  // the launch for the other rows takes SMs as they get free
  if (tid == 0) sh.count = 0;
  int rows = a.B;
  if constexpr (!WHOLE) {  // list this kernel's rows
    rows = 0;
    for (int r0 = 0; r0 < a.B; r0 += WIDTH) {
      const int r = r0 + tid;
      const float temperature = r < a.B ? a.temperature[r] : 0.f;
      const bool mine = r < a.B && ordinary(temperature) && cuts_nothing(a.top_k[r], a.top_p[r], a.min_p[r], a.V);
      const uint32_t same = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) sh.counts[warp] = __popc(same);
      __syncthreads();
      const uint32_t count = sh.counts[lane];
      const int before = (int)__reduce_add_sync(0xffffffffu, lane < warp ? count : 0u);
      if (mine) listed[rows + before + __popc(same & ((1u << lane) - 1))] = Listed{r, temperature};
      rows += (int)__reduce_add_sync(0xffffffffu, count);
      __syncthreads();
    }
  }
  // a row spans at most 17 blocks: fewer than a warp's lanes, which merge its parts
  const int line = rows * pieces, per_block = max((int)(((uint32_t)line + gridDim.x - 1) / gridDim.x), (pieces + 15) / 16);
  const int from = (int)min((long long)line, (long long)per_block * blockIdx.x);
  if (from >= line) return;
  const int to = min(line - from, per_block) + from;

  // A stretch of a row: pieces i ... end - 1, of which the whole ones (all tokens inside the row) are copied.
  struct Stretch {
    int at, row, i, end, skew;  // at: on the line
  };
  const auto row_logits = [&](int row) { return static_cast<const T*>(a.logits) + row * a.row_stride; };
  const auto row_noise = [&](int row) { return a.noise + row * a.noise_stride; };
  const auto stretch_at = [&](int at, int i) {
    const int row = WHOLE ? at : listed[at].row;
    return Stretch{at, row, i, min(pieces, to - at * pieces), (int)((reinterpret_cast<uintptr_t>(row_logits(row)) % 16) / sizeof(T))};
  };
  const auto last_one = [&](const Stretch& s) { return s.at * pieces + s.end == to; };

  const int first_row = from / pieces;
  Stretch use = stretch_at(first_row, from - first_row * pieces);
  // What is loaded next, of this thread.
  Stretch ahead = use;
  const T* next_logits;
  const float* next_noise;  // of the warp's first piece
  int next, next_from, next_to;  // piece, and the bounds of those to load
  bool more = true, together = true;
  const auto open = [&] {
    next = ahead.i + tid;
    next_from = ahead.skew > 0;
    next_to = min((ahead.skew + a.V) / E, ahead.end);
    next_logits = row_logits(ahead.row) + (next * E - ahead.skew);
    next_noise = row_noise(ahead.row) + ((next - lane) * E - ahead.skew);
    together = reinterpret_cast<uintptr_t>(next_noise) % 16 == 0;
  };
  open();
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring), luck_addr = (uint32_t)__cvta_generic_to_shared(lucks);
  const auto issue = [&](int stage) {
    if (more) {
      const uint32_t slot = ring_addr + stage * (UNITS * WIDTH * 16);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const auto wanted = [&](int piece) {  // of the warp
          const int i = next - lane + j * WIDTH + piece;
          return i >= next_from && i < next_to;
        };
        if (wanted(lane)) copy16(slot + j * WIDTH * 16, next_logits + j * WIDTH * E);
        if constexpr (!GREEDY) {
          const float* const luck = next_noise + j * WIDTH * E;
          const uint32_t there = luck_addr + stage * (UNITS * WIDTH * 16) + j * WIDTH * E * 4;
          if (together) {
#pragma unroll
            for (int x = lane; x < 8 * E; x += 32)
              if (wanted(x / (E / 4))) copy16(there + x * 16, luck + x * 4);
          } else {
#pragma unroll 1
            for (int x = lane; x < 32 * E; x += 32)
              if (wanted(x / E)) copy4(there + x * 4, luck + x);
          }
        }
      }
      next += TURN;
      next_logits += TURN * E;
      next_noise += TURN * E;
      ahead.i += TURN;
      if (ahead.i >= ahead.end) {
        more = !last_one(ahead);
        if (more) {
          ahead = stretch_at(ahead.at + 1, 0);
          open();
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // Of the warp: the reference, and the best score so far (greedy: logit) with its token.  w / e > score is asked as
  // w > score e, without a division; of a warp's tokens only some ten per row get past that.
  float nothing;  // the reference where no token has been seen that can be drawn: their logits lie above -1e30
  float reference, score;
  uint32_t drawn;
  Pair sums;  // of the thread
  const auto clear = [&] {
    if constexpr (!WHOLE) {
      const float temperature = listed[use.at].temperature, most = 1.4426950216293335f;  // of log2(e)
      hi = most / temperature;
      lo = (fmaf(-hi, temperature, most) + 1.925963033500011e-8f) / temperature;
    }
    nothing = -1e30f * hi;
    reference = nothing;
    score = GREEDY ? -1e30f : -1.f;
    drawn = NOBODY;
    sums = pair(0.f, 0.f);
  };
  clear();
  // Anything but a number of 0 or more counts as the largest: such a token loses.
  const auto sane = [](float e) { return __uint_as_float(min(__float_as_uint(e), 0x7f7fffffu)); };

#pragma unroll 1
  for (int s = 0; s < STAGES - 1; ++s) issue(s);
  int parity = 0, merger = 0;
  for (int stage = 0;; stage = (stage + 1) % STAGES) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();  // a warp reads what it copied itself
    issue((stage + STAGES - 1) % STAGES);
    if (use.i + warp * 32 < use.end) {
      const int first = (use.i + tid) * E - use.skew, whole_from = use.skew > 0, whole_to = (use.skew + a.V) / E;
      const uint4* const slot = ring + stage * UNITS * WIDTH;
      float l[8];
      [[maybe_unused]] float luck[8];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = use.i + j * WIDTH + tid;
        uint4 raw = make_uint4(none, none, none, none);
#pragma unroll
        for (int e = 0; e < E; ++e) luck[j * E + e] = 1.f;
        if (i < use.end) {
          if (i >= whole_from && i < whole_to) {
            raw = slot[j * WIDTH];
            if constexpr (!GREEDY) {
#pragma unroll
              for (int x = 0; x < E / 4; ++x) {
                const float4 e = *reinterpret_cast<const float4*>(lucks + stage * (UNITS * WIDTH * 4) + j * WIDTH * E + lane * E + 4 * x);
                luck[j * E + 4 * x] = e.x, luck[j * E + 4 * x + 1] = e.y, luck[j * E + 4 * x + 2] = e.z, luck[j * E + 4 * x + 3] = e.w;
              }
            }
          } else {  // at one of the row's ends: the tokens that belong to it
            uint32_t u[4] = {none, none, none, none};
            const T* const logits = row_logits(use.row);
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int token = first + j * WIDTH * E + e;
              if (token < 0 || token >= a.V) continue;
              if constexpr (sizeof(T) == 4) u[e] = __float_as_uint(logits[token]);
              else u[e / 2] = (u[e / 2] & (e % 2 ? 0xffffu : 0xffff0000u)) | ((uint32_t)__bfloat16_as_ushort(logits[token]) << (16 * (e % 2)));
              if constexpr (!GREEDY) luck[j * E + e] = row_noise(use.row)[token];
            }
            raw = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
        const Piece<T> p(raw);
#pragma unroll
        for (int x = 0; x < E; ++x) l[j * E + x] = fmaxf(p.v[x], -1e30f);  // -inf and NaN: no weight at any ordinary temperature
      }
      float top = -1e30f;
#pragma unroll
      for (int x = 0; x < 8; ++x) top = fmaxf(top, l[x]);
      const auto token_at = [&](int x) { return (uint32_t)(first + (E == 4 ? x / 4 * (WIDTH * E) + x % 4 : x)); };
      if (__any_sync(0xffffffffu, GREEDY ? top > score : top * hi > reference)) {
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float higher = fmaxf(reference, ceilf(top * hi)), scale = fast_exp2(reference - higher);
        sums = times(sums, pair(scale, scale));
        reference = higher;
        if constexpr (GREEDY) {
          uint32_t token = NOBODY;
#pragma unroll
          for (int x = 7; x >= 0; --x) token = l[x] == top ? token_at(x) : token;
          score = top;
          drawn = __reduce_min_sync(0xffffffffu, token);
        } else if (score > 0.f) {
          score *= scale;
        }
      }
      if (reference > nothing) {
        float w[8];
        bool wins = false;
#pragma unroll
        for (int x = 0; x < 8; x += 2) {
          const Pair both = pair(l[x], l[x + 1]);
          const Pair z = fma(both, pair(lo, lo), fma(both, pair(hi, hi), pair(-reference, -reference)));
          w[x] = fast_exp2(low(z));
          w[x + 1] = fast_exp2(high(z));
          sums = plus(sums, pair(w[x], w[x + 1]));
          if constexpr (!GREEDY) {
            const Pair least = times(pair(score, score), pair(luck[x], luck[x + 1]));
            wins = wins || w[x] > low(least) || w[x + 1] > high(least);
          }
        }
        if constexpr (!GREEDY) {
          if (__any_sync(0xffffffffu, wins)) {
            uint32_t key = 0u, token = NOBODY;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const uint32_t k = l[x] > -1e30f ? key_of(__fdividef(w[x], sane(luck[x]))) : 0u;
              if (k > key) {
                key = k;
                token = token_at(x);
              }
            }
            const uint32_t best = __reduce_max_sync(0xffffffffu, key);
            if (best > key_of(score)) {  // tokens of later turns have higher indices: among equals the first stays
              score = value_of(best);
              drawn = __reduce_min_sync(0xffffffffu, key == best ? token : NOBODY);
            }
          }
        }
      }
    }
    use.i += TURN;
    if (use.i < use.end) continue;

    // ---- the stretch ends
    float sum = low(sums) + high(sums);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.parts[parity][warp] = Part{reference, sum, drawn == NOBODY ? 0u : key_of(score), drawn};
    __syncthreads();  // the other half of `parts` was read before its readers came here
    if (warp == merger) {
      const int row_from = use.at * pieces;
      bool complete = row_from >= from && row_from + pieces <= to;
      const Part* list = sh.parts[parity];
      int n = GROUPS, step = 1, skip = 0;
      for (;;) {
        Part mine{-INFINITY, 0.f, 0u, NOBODY};
        if (lane < n) mine = load(list + lane * step + (lane == 0 ? skip : 0));
        float most = mine.reference;
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float down = fast_exp2(mine.reference - most);
        uint32_t key = GREEDY ? mine.key : key_of(value_of(mine.key) * down), token = mine.token;
        float total = mine.sum * down;
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const uint32_t first = __reduce_max_sync(0xffffffffu, key);
        token = __reduce_min_sync(0xffffffffu, key == first ? token : NOBODY);
        key = first;
        if (complete) {
          if (lane == 0) {
            // beyond this the products with the rate lose the differences (or a logit is infinite)
            if (fabsf(most) < 1e5f && token != NOBODY) {
              const float l = Piece<T>::one(row_logits(use.row)[token]);
              a.token[use.row] = token;
              a.logprob[use.row] = (fmaf(l, lo, fmaf(l, hi, -most)) - __log2f(total)) * LN2;
            } else {
              sh.rows[sh.count++] = use.row;
            }
          }
          break;
        }
        const int first_block = row_from / per_block, last_block = (row_from + pieces - 1) / per_block;
        Part* const all = reinterpret_cast<Part*>(a.partial);
        bool last = false;
        if (lane == 0) {
          all[2 * blockIdx.x + (row_from > from)] = Part{most, total, key, token};
          last = arrive(a.arrived + first_block) == (unsigned)(last_block - first_block);
          if (last) a.arrived[first_block] = 0;
        }
        if (!__any_sync(0xffffffffu, last)) break;
        __syncwarp();
        list = all + 2 * first_block;
        n = last_block - first_block + 1;
        step = 2;
        skip = row_from > per_block * first_block;
        complete = true;
      }
    }
    if (last_one(use)) break;
    use = stretch_at(use.at + 1, 0);
    clear();
    parity ^= 1;
    merger = (merger + 1) % GROUPS;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- rows whose logits are too large for a rate without a reference, or infinite, and rows without a token to draw
  __syncthreads();
  for (int x = 0; x < sh.count; ++x) {
    const int row = sh.rows[x];
    const T* const logits = static_cast<const T*>(a.logits) + row * a.row_stride;
    const float* const noise = a.noise + row * a.noise_stride;
    uint32_t best = 0u;
#pragma unroll 4
    for (int token = tid; token < a.V; token += WIDTH) best = max(best, key_of(Piece<T>::one(logits[token])));
    best = (uint32_t)block_reduce<GROUPS>((unsigned long long)best, sh.picks, [](unsigned long long v, unsigned long long w) { return max(v, w); });
    if (best == 0u) {
      if (tid == 0) {
        a.token[row] = -1;
        a.logprob[row] = -INFINITY;
      }
      continue;
    }
    const Weights weight(value_of(best), GREEDY ? 1.f : a.temperature[row]);
    double total = 0.0;
    unsigned long long pick = 0;
    for (int token = tid; token < a.V; token += WIDTH) {
      const float l = Piece<T>::one(logits[token]);
      const uint32_t key = key_of(l);
      if (key == 0u) continue;
      const float w = weight(l);
      total += (double)w;
      const uint32_t score = GREEDY ? key : key_of(__fdividef(w, sane(noise[token])));
      pick = max(pick, ((unsigned long long)score << 32) | (0xffffffffu - (uint32_t)token));
    }
    total = block_reduce<GROUPS>(total, sh.sums, [](double v, double w) { return v + w; });
    pick = block_reduce<GROUPS>(pick, sh.picks, [](unsigned long long v, unsigned long long w) { return max(v, w); });
    if (tid == 0) {
      const int token = (int)(0xffffffffu - (uint32_t)pick);
      a.token[row] = token;
      a.logprob[row] = (weight.exponent(Piece<T>::one(logits[token])) - __log2f((float)total)) * LN2;
    }
  }
}

}  // namespace

template <bool GREEDY, bool WHOLE, typename T>
static cudaError_t stream_as(const Args& a, int sms, cudaStream_t stream) {
  using R = Ring<GREEDY, T>;
  const int pieces = (a.V + 2 * R::E - 2) / R::E, fixed = R::BYTES + (int)sizeof(Small);
  // dynamic shared memory beyond 48 KB is opted into once per device
  static unsigned long long opted = 0;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  const unsigned long long bit = 1ull << (device & 63);
  if (!(__atomic_load_n(&opted, __ATOMIC_ACQUIRE) & bit)) {
    err = cudaFuncSetAttribute(stream_kernel<GREEDY, WHOLE, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               fixed + (WHOLE ? 0 : kMostListed * (int)sizeof(Listed)));
    if (err != cudaSuccess) return err;
    __atomic_fetch_or(&opted, bit, __ATOMIC_RELEASE);
  }
  const double rate = 1.4426950408889634 / (GREEDY ? 1.0 : (double)a.temperature.same);
  const float hi = (float)rate, lo = (float)(rate - (double)hi);
  stream_kernel<GREEDY, WHOLE, T><<<(unsigned)sms, WIDTH, fixed + (WHOLE ? 0 : a.B * (int)sizeof(Listed)), stream>>>(a, pieces, hi, lo);
  return cudaGetLastError();
}

cudaError_t launch_stream(const Args& a, bool whole, int sms, cudaStream_t stream) {
  if (!whole) return a.wide ? stream_as<false, false, float>(a, sms, stream) : stream_as<false, false, __nv_bfloat16>(a, sms, stream);
  if (a.temperature.same > 0.f) return a.wide ? stream_as<false, true, float>(a, sms, stream) : stream_as<false, true, __nv_bfloat16>(a, sms, stream);
  return a.wide ? stream_as<true, true, float>(a, sms, stream) : stream_as<true, true, __nv_bfloat16>(a, sms, stream);
}

long long workspace_floats(int sms) { return 2ll * sms * (long long)(sizeof(Part) / sizeof(float)); }
int workspace_counters(int sms) { return sms; }

}  // namespace sampling
}  // namespace ht
