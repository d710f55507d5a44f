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
// Each cut is found by bisection over the bits of the ordered logit: 32 passes over the row that count
// the tokens, or sum the weights, at or above a pivot.
#include "generation.cuh"

namespace ht {
namespace sampling {

constexpr int THREADS = 1024;
constexpr float LOG2E = 1.4426950408889634f;

// Unsigned keys in the order of the floats; NaN and -inf share the lowest key.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(l + 0.f);  // -0 + 0 = +0: equal logits have equal keys
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return key == 0u ? -INFINITY : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <typename T>
__device__ __forceinline__ float load(const void* p, long long i) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else return static_cast<const float*>(p)[i];
}

// w = exp((l - best) / T), the quotient log2(e) / T carried in two floats.
struct Weights {
  float best, hi, lo;
  __device__ __forceinline__ float exponent(float l) const {
    if (l == best) return 0.f;
    const float d = l - best;
    if (!(d > -INFINITY)) return -INFINITY;
    const float y = d * hi;  // the correction only where it is finite and the weight is not zero anyway
    return y > -1024.f ? fmaf(d, hi, d * lo) : y;
  }
  __device__ __forceinline__ float operator()(float l) const { return exp2f(exponent(l)); }
};

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* scratch, Op op) {
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
  __syncthreads();
  v = scratch[threadIdx.x % 32];
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(Args a) {
  __shared__ float fs[32];
  __shared__ uint32_t us[32];
  __shared__ unsigned long long ls[32];
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* logits = static_cast<const T*>(a.logits) + row * a.row_stride;
  const auto sum = [](float x, float y) { return x + y; };
  const auto add = [](uint32_t x, uint32_t y) { return x + y; };
  const auto most = [](uint32_t x, uint32_t y) { return max(x, y); };

  uint32_t best_key = 0;
  for (int i = tid; i < a.V; i += THREADS) best_key = max(best_key, key_of(load<T>(logits, i)));
  best_key = block_reduce(best_key, us, most);
  if (best_key == 0u) {
    if (tid == 0) {
      a.token[row] = -1;
      a.logprob[row] = -INFINITY;
    }
    return;
  }
  const float temperature = a.temperature[row];
  const bool greedy = !(temperature > 0.f);
  const double rate = 1.4426950408889634 / (greedy ? 1.0 : (double)temperature);
  Weights weight{value_of(best_key), (float)rate, 0.f};
  weight.lo = isinf(weight.hi) ? 0.f : (float)(rate - (double)weight.hi);

  float total = 0.f;
  for (int i = tid; i < a.V; i += THREADS) total += weight(load<T>(logits, i));
  total = block_reduce(total, fs, sum);

  // Tokens with key > cut stay, and those with key == cut and one of the first `ties` indices among them.
  uint32_t cut = 0, ties = 0xffffffffu;
  const int top_k = a.top_k[row];
  const float top_p = a.top_p[row];
  if (!greedy) {
    const auto count_from = [&](uint32_t pivot) {
      uint32_t c = 0;
      for (int i = tid; i < a.V; i += THREADS) c += key_of(load<T>(logits, i)) >= pivot;
      return block_reduce(c, us, add);
    };
    const auto mass_from = [&](uint32_t pivot) {
      float m = 0.f;
      for (int i = tid; i < a.V; i += THREADS) {
        const float l = load<T>(logits, i);
        if (key_of(l) >= pivot) m += weight(l);
      }
      return block_reduce(m, fs, sum);
    };
    float mass = total;
    if (top_k > 0 && top_k < a.V) {
      for (int bit = 31; bit >= 0; --bit)  // the largest key that top_k tokens reach
        if (count_from(cut | (1u << bit)) >= (uint32_t)top_k) cut |= 1u << bit;
      const uint32_t above = cut == 0xffffffffu ? 0u : count_from(cut + 1);
      ties = top_k - above;
      mass = (cut == 0xffffffffu ? 0.f : mass_from(cut + 1)) + ties * weight(value_of(cut));
    }
    if (!(top_p >= 1.f)) {
      const float limit = top_p * mass;
      uint32_t low = 0;
      for (int bit = 31; bit >= 0; --bit)  // the largest key at which the mass above and at it reaches the limit
        if (mass_from(low | (1u << bit)) >= limit) low |= 1u << bit;
      low = min(low, best_key);
      const float above = low == 0xffffffffu ? 0.f : mass_from(low + 1), w = weight(value_of(low));
      const uint32_t equal = count_from(low) - (low == 0xffffffffu ? 0u : count_from(low + 1));
      uint32_t n = 0;  // the first n of the equal ones have less than the limit before them
      for (uint32_t bit = 1u << 30; bit > 0; bit >>= 1)
        if ((n | bit) <= equal && above + ((n | bit) - 1) * w < limit) n |= bit;
      if (low > cut || (low == cut && n < ties)) {
        cut = low;
        ties = n;
      }
    }
  }
  if (greedy || (cut == best_key && ties == 0u)) {
    cut = best_key;
    ties = 1;
  }
  // The index of the last tie that stays: bisection over the indices.
  uint32_t last = a.V - 1;
  {
    uint32_t equal = 0;
    for (int i = tid; i < a.V; i += THREADS) equal += key_of(load<T>(logits, i)) == cut;
    equal = block_reduce(equal, us, add);
    if (equal > ties) {
      uint32_t low = 0, high = a.V - 1;
      while (low < high) {
        const uint32_t mid = (low + high) / 2;
        uint32_t c = 0;
        for (uint32_t i = tid; i <= mid; i += THREADS) c += key_of(load<T>(logits, i)) == cut;
        c = block_reduce(c, us, add);
        if (c >= ties) high = mid;
        else low = mid + 1;
      }
      last = low;
    }
  }
  const float min_p = a.min_p[row];
  const float* noise = a.noise + row * a.noise_stride;
  // (score, lowest index) as one ordered number
  unsigned long long winner = 0;
  for (int i = tid; i < a.V; i += THREADS) {
    const float l = load<T>(logits, i);
    const uint32_t key = key_of(l);
    if (key == 0u || key < cut || (key == cut && (uint32_t)i > last)) continue;
    const float w = weight(l);
    if (key != best_key && !(w >= min_p)) continue;
    const float score = __fdiv_rn(w, noise[i]);
    // a NaN (from a random number that is none) ranks below every score, but still names a token
    winner = max(winner, ((unsigned long long)max(key_of(score), 1u) << 32) | (0xffffffffu - (uint32_t)i));
  }
  winner = block_reduce(winner, ls, [](unsigned long long x, unsigned long long y) { return max(x, y); });
  if (tid == 0) {
    const uint32_t token = 0xffffffffu - (uint32_t)winner;
    a.token[row] = token;
    a.logprob[row] = weight.exponent(load<T>(logits, token)) * 0.6931471805599453f - logf(total);
  }
}

cudaError_t launch(const Args& a, int sms, cudaStream_t stream) {
  if (a.wide) sample_kernel<float><<<(unsigned)a.B, THREADS, 0, stream>>>(a);
  else sample_kernel<__nv_bfloat16><<<(unsigned)a.B, THREADS, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace sampling
}  // namespace ht
