// Writing keys and values into a paged cache, and reading them back.
//
// A layer's pool is [pages, Hkv, page_size, D] for the keys and the same for the values; slot s is
// row s % page_size of page s / page_size.  The pool holds bf16 rows, or rows of 8-bit values q
// (int8, or fp8 e4m3) with one fp32 scale per token and head:
//     scale = max(amax(|x|) * fl(1/Q), 2^-64),   q = rn(x * fl(1/scale)),   x' = bf16(q * scale)
// with Q = 127 (int8) or 448 (e4m3).  One scale per row: a row is written once, by the token that
// owns it, so nothing that is already in the cache has to be rescaled.  Every step is one IEEE
// operation (the build's fast-math division is avoided), so the stored bytes do not depend on who
// computes them.  The floor on the scale keeps fl(1/scale) finite for rows of zeros; a row with an
// infinity or a NaN gets a NaN scale, so that it reads back as NaN instead of as a plausible value.
//
// Bound: memory; every byte is touched once.  A row takes D / 8 lanes with 16 bytes of bf16 each; a thread has
// its place of the keys and of the values in flight together: 16384 tokens of 8 x 128 are written and read back in 35.8 us.
// (Two or four rows a thread measured 40 and 41 us where this took 37, before the maxima were packed, and up to twice the time
// on 32 tokens, where there are then fewer warps than schedulers.)  Integers are converted with additions of a power of two and byte permutes: the conversion
// instructions run at an eighth of their rate and would bind before the memory does.
#include "generation.cuh"

namespace ht {
namespace kv {

constexpr int THREADS = 256;

// Division of row numbers (below 2^31) by the number of heads: the high half of a product, shifted.
struct Divider {
  uint32_t by, factor;
  int shift;  // -1: by one
  explicit Divider(int d) : by((uint32_t)d) {
    int log = 0;
    while ((1ll << log) < d) ++log;
    shift = log - 1;
    factor = (uint32_t)((1ull << (31 + log)) / (unsigned)d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t r) const { return shift < 0 ? r : __umulhi(r, factor) >> shift; }
};

__device__ __forceinline__ long long slot_of(const void* slots, int wide, int t) {
  return wide ? static_cast<const long long*>(slots)[t] : (long long)static_cast<const int*>(slots)[t];
}

// Row of the pool that holds head h of `slot`, or -1 for a slot outside it.
__device__ __forceinline__ long long pool_row(const Pool& p, long long slot, int h) {
  if (slot < 0 || slot >= p.pages << p.page_shift) return -1;
  return (((slot >> p.page_shift) * p.Hkv + h) << p.page_shift) + (slot & ((1ll << p.page_shift) - 1));
}

// rn(x * inv) of 8 values as bytes.  |x * inv| is at most Q (1 + 2^-22), which rounds to Q: nothing has to be cut off.
template <int F>
__device__ __forceinline__ uint2 quantise8(const float* x, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (F == kInt8) {
      // 1.5 * 2^23 + y has a last place of 1: the sum is rounded to the nearest integer, whose low byte is the value
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(x[4 * h + j], inv), 12582912.f));
      w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[4 * h], inv), __fmul_rn(x[4 * h + 1], inv)), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi =
          __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(x[4 * h + 2], inv), __fmul_rn(x[4 * h + 3], inv)), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | (hi << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

// The four values of a word.
template <int F>
__device__ __forceinline__ float4 values_of(uint32_t w) {
  if constexpr (F == kInt8) {
    const uint32_t u = w ^ 0x80808080u;  // value + 128 as an unsigned byte; 2^23 + byte is a float with that byte at its end
    const auto one = [&](uint32_t pick) { return __fadd_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, pick)), -8388736.f); };
    return make_float4(one(0x7440), one(0x7441), one(0x7442), one(0x7443));
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 x = __half22float2(__half2(a)), y = __half22float2(__half2(b));
    return make_float4(x.x, x.y, y.x, y.y);
  }
}

template <int F, int D>
__global__ void __launch_bounds__(THREADS) write_kernel(const __grid_constant__ WriteArgs a, const Divider heads) {
  constexpr int LANES = D / 8, PER_BLOCK = THREADS / LANES;
  const int rows = (int)a.T * a.pool.Hkv, lane = threadIdx.x % LANES;
  // every lane of a warp makes the same number of turns, so the shuffles below always see a full warp
  for (int base = blockIdx.x * PER_BLOCK; base < rows; base += gridDim.x * PER_BLOCK) {
    const int r = base + threadIdx.x / LANES;
    uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    long long at = -1;
    if (r < rows) {
      const int t = (int)heads((uint32_t)r), h = r - t * a.pool.Hkv;
      raw[0] = __ldcs(reinterpret_cast<const uint4*>(a.src[0] + t * a.tok[0] + h * a.head[0] + lane * 8));
      raw[1] = __ldcs(reinterpret_cast<const uint4*>(a.src[1] + t * a.tok[1] + h * a.head[1] + lane * 8));
      at = pool_row(a.pool, slot_of(a.slots, a.wide, t), h);
    }
    if constexpr (F == kBf16) {
      if (at >= 0) {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.pool.k) + at * D + lane * 8) = raw[0];
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.pool.v) + at * D + lane * 8) = raw[1];
      }
    } else {
      // The rows' largest magnitudes as 16 bits each (NaN > infinity > every finite value), the key's and the value's side by
      // side through one reduction.
      uint32_t top[2];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t m = 0x7fff7fffu;
        top[which] = __vmaxu2(__vmaxu2(raw[which].x & m, raw[which].y & m), __vmaxu2(raw[which].z & m, raw[which].w & m));
      }
      uint32_t both = __vmaxu2(__byte_perm(top[0], top[1], 0x5410), __byte_perm(top[0], top[1], 0x7632));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float largest = __uint_as_float(which ? both & 0xffff0000u : both << 16);
        const bool finite = largest < INFINITY;
        const float scale =
            finite ? fmaxf(__fmul_rn(largest, F == kInt8 ? 1.0f / 127.0f : 1.0f / 448.0f), kMinScale) : __int_as_float(0x7fc00000);
        const uint32_t u[4] = {raw[which].x, raw[which].y, raw[which].z, raw[which].w};
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[2 * j] = __uint_as_float(u[j] << 16);
          x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
        uint2 q = quantise8<F>(x, __frcp_rn(scale));
        if (!finite) q = make_uint2(0, 0);
        if (at >= 0) {
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(which ? a.pool.v : a.pool.k) + at * D + lane * 8) = q;
          if (lane == 0) (which ? a.pool.v_scale : a.pool.k_scale)[at] = scale;
        }
      }
    }
  }
}

template <int F, int D>
__global__ void __launch_bounds__(THREADS) read_kernel(const __grid_constant__ ReadArgs a, const Divider heads) {
  constexpr int LANES = D / 8, PER_BLOCK = THREADS / LANES;
  const int rows = (int)a.T * a.pool.Hkv, lane = threadIdx.x % LANES;
  for (int r = blockIdx.x * PER_BLOCK + threadIdx.x / LANES; r < rows; r += gridDim.x * PER_BLOCK) {
    const int t = (int)heads((uint32_t)r), h = r - t * a.pool.Hkv;
    const long long at = pool_row(a.pool, slot_of(a.slots, a.wide, t), h);
    uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    float scale[2] = {0.f, 0.f};
    if (at >= 0) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const void* const pool = which ? a.pool.v : a.pool.k;
        if constexpr (F == kBf16) {
          raw[which] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(pool) + at * D + lane * 8);
        } else {
          const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at * D + lane * 8);
          raw[which].x = q.x;
          raw[which].y = q.y;
          scale[which] = (which ? a.pool.v_scale : a.pool.k_scale)[at];
        }
      }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint4 out = raw[which];
      if constexpr (F != kBf16) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float4 x = values_of<F>(j ? raw[which].y : raw[which].x);
          const __nv_bfloat162 p = __floats2bfloat162_rn(__fmul_rn(x.x, scale[which]), __fmul_rn(x.y, scale[which]));
          const __nv_bfloat162 q = __floats2bfloat162_rn(__fmul_rn(x.z, scale[which]), __fmul_rn(x.w, scale[which]));
          w[2 * j] = *reinterpret_cast<const uint32_t*>(&p);
          w[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&q);
        }
        out = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __stcs(reinterpret_cast<uint4*>(a.dst[which] + t * a.tok[which] + h * a.head[which] + lane * 8), out);
    }
  }
}

static unsigned row_blocks(long long rows, int D, int sms) {
  const long long per_block = THREADS / (D / 8), blocks = (rows + per_block - 1) / per_block;
  return (unsigned)(blocks < sms * 16ll ? blocks : sms * 16ll);
}

cudaError_t launch_write(const WriteArgs& a, int sms, cudaStream_t stream) {
  const unsigned blocks = row_blocks(a.T * a.pool.Hkv, a.pool.D, sms);
  by_format(a.pool, [&](auto f, auto d) { write_kernel<decltype(f)::value, decltype(d)::value><<<blocks, THREADS, 0, stream>>>(a, Divider(a.pool.Hkv)); });
  return cudaGetLastError();
}

cudaError_t launch_read(const ReadArgs& a, int sms, cudaStream_t stream) {
  const unsigned blocks = row_blocks(a.T * a.pool.Hkv, a.pool.D, sms);
  by_format(a.pool, [&](auto f, auto d) { read_kernel<decltype(f)::value, decltype(d)::value><<<blocks, THREADS, 0, stream>>>(a, Divider(a.pool.Hkv)); });
  return cudaGetLastError();
}

}  // namespace kv
}  // namespace ht
