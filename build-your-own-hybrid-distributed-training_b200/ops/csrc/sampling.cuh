// What the sampling kernels share: orders of floats, weights and their sums, rows in pieces of 16 bytes.
#pragma once

#include "generation.cuh"

namespace ht {
namespace sampling {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr float LN2 = 0.6931471805599453f;
constexpr float MASS = 0x1p44f;  // what a weight of 1 is held as

// Unsigned keys in the order of the floats; -inf has the lowest one.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(l + 0.f);  // -0 + 0 = +0: equal logits have equal keys
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {  // keys below that of the lowest number stand for -inf
  return key <= 0x007fffffu ? -INFINITY : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in a register pair, on which one instruction works.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
  return p;
}
__device__ __forceinline__ float low(Pair p) { return __uint_as_float((uint32_t)p); }
__device__ __forceinline__ float high(Pair p) { return __uint_as_float((uint32_t)(p >> 32)); }
__device__ __forceinline__ Pair plus(Pair x, Pair y) {
  Pair p;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(p) : "l"(x), "l"(y));
  return p;
}
__device__ __forceinline__ Pair times(Pair x, Pair y) {
  Pair p;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(p) : "l"(x), "l"(y));
  return p;
}
__device__ __forceinline__ Pair fma(Pair x, Pair y, Pair z) {
  Pair p;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(p) : "l"(x), "l"(y), "l"(z));
  return p;
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
  __device__ __forceinline__ Pair operator()(Pair l) const {  // the same, but not if `single`
    const Pair d = plus(l, pair(-best, -best));
    const Pair x = fma(d, pair(hi, hi), times(pair(fmaxf(low(d), least), fmaxf(high(d), least)), pair(lo, lo)));
    return pair(fast_exp2(low(x)), fast_exp2(high(x)));
  }
  // Masses as integers, which add up to the same in every order: multiples of 2^-44, and, for weights that are known to be at
  // most 2^-k, of 2^-(31 + k) in half as many bits.
  __device__ __forceinline__ unsigned long long mass(float l) const { return __float2ull_rn((*this)(l)*MASS); }
  __device__ __forceinline__ uint32_t mass(float l, int k) const { return __float2uint_rn((*this)(l)*__uint_as_float((uint32_t)(127 + 31 + k) << 23)); }
};

// A sum of weights, two at a time, that comes out the same in every order (and so for every alignment of the row): multiples
// of 2^-16, which a thread's few hundred terms add without rounding, and what they leave of each weight (at most 2^-17),
// whose roundings lie far below the fp32 result.
struct Sums {
  Pair coarse = pair(0.f, 0.f), fine = pair(0.f, 0.f);
  __device__ __forceinline__ void add(Pair w) {
    const Pair near = plus(plus(w, pair(128.f, 128.f)), pair(-128.f, -128.f));
    coarse = plus(coarse, near);
    fine = plus(fine, fma(near, pair(-1.f, -1.f), w));
  }
  __device__ __forceinline__ double value() const { return ((double)low(coarse) + (double)high(coarse)) + (double)(low(fine) + high(fine)); }
};

template <int N = WARPS, typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* scratch, Op op) {  // of a block of N warps
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
  __syncthreads();
  v = scratch[threadIdx.x % N];
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// Rows that sampling_stream.cu takes: nothing is cut, and the temperature is an ordinary one.
__host__ __device__ inline bool cuts_nothing(int top_k, float top_p, float min_p, int V) {
  return (top_k <= 0 || top_k >= V) && top_p >= 1.f && min_p <= 0.f;  // false for NaN
}
__host__ __device__ inline bool ordinary(float temperature) { return temperature > 1e-3f && temperature < 1e3f; }

}  // namespace sampling
}  // namespace ht
