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
// Bound: memory.  Both kernels touch every byte once, 16 bytes of bf16 per lane and D / 8 lanes per
// row.
#include "generation.cuh"

namespace ht {
namespace kv {

constexpr int THREADS = 256;

template <int F>
__device__ __forceinline__ uint2 quantise8(const float* x, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float y = __fmul_rn(x[4 * h + j], inv);
      if constexpr (F == kInt8) {
        b[j] = (uint32_t)max(-127, min(127, __float2int_rn(y))) & 0xffu;
      } else {
        b[j] = __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
      }
    }
    w[h] = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
  }
  return make_uint2(w[0], w[1]);
}

template <int F>
__device__ __forceinline__ float value_of(uint32_t byte) {
  if constexpr (F == kInt8) return (float)(int8_t)byte;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

__device__ __forceinline__ long long slot_of(const void* slots, int wide, long long t) {
  return wide ? static_cast<const long long*>(slots)[t] : (long long)static_cast<const int*>(slots)[t];
}

// Row index (in rows of D) of `slot` for head h in a [pages, Hkv, page_size, D] pool.
__device__ __forceinline__ long long pool_row(long long slot, int h, int Hkv, int page_shift) {
  const long long page = slot >> page_shift;
  return ((page * Hkv + h) << page_shift) + (slot & ((1ll << page_shift) - 1));
}

template <int F, int D>
__global__ void __launch_bounds__(THREADS) write_kernel(WriteArgs a) {
  constexpr int LANES = D / 8;
  const long long rows = a.T * a.pool.Hkv;
  const int lane = threadIdx.x % LANES;
  const int which = blockIdx.y;  // 0: keys, 1: values
  const __nv_bfloat16* const src = which ? a.src[1] : a.src[0];
  const long long tok = which ? a.tok[1] : a.tok[0], head = which ? a.head[1] : a.head[0];
  void* const pool = which ? a.pool.v : a.pool.k;
  float* const scales = which ? a.pool.v_scale : a.pool.k_scale;
  const long long step = (long long)gridDim.x * (THREADS / LANES);
  const long long first = (long long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
  // every lane of a warp makes the same number of turns, so the shuffles below always see a full warp
  for (long long base = first; base - threadIdx.x / LANES < rows; base += step) {
    const bool on = base < rows;
    const long long t = on ? base / a.pool.Hkv : 0;
    const int h = on ? (int)(base - t * a.pool.Hkv) : 0;
    const long long slot = on ? slot_of(a.slots, a.wide, t) : -1;
    const bool stored = slot >= 0 && slot < a.pool.pages << a.pool.page_shift;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (stored) raw = *reinterpret_cast<const uint4*>(src + t * tok + h * head + lane * 8);
    const long long row = stored ? pool_row(slot, h, a.pool.Hkv, a.pool.page_shift) : 0;
    if constexpr (F == kBf16) {
      if (stored) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(pool) + row * D + lane * 8) = raw;
    } else {
      const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
      float x[8];
      uint32_t top = 0;  // the largest magnitude as bits: NaN > infinity > every finite value
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(u[j] << 16);
        x[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        top = max(top, max((u[j] << 16) & 0x7fffffffu, u[j] & 0x7fff0000u));
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const bool finite = top < 0x7f800000u;
      const float scale = finite ? fmaxf(__fmul_rn(__uint_as_float(top), F == kInt8 ? 1.0f / 127.0f : 1.0f / 448.0f), kMinScale)
                                 : __int_as_float(0x7fc00000);
      const uint2 q = finite ? quantise8<F>(x, __frcp_rn(scale)) : make_uint2(0, 0);
      if (stored) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + row * D + lane * 8) = q;
        if (lane == 0) scales[row] = scale;
      }
    }
  }
}

template <int F, int D>
__global__ void __launch_bounds__(THREADS) read_kernel(ReadArgs a) {
  constexpr int LANES = D / 8;
  const long long rows = a.T * a.pool.Hkv;
  const int lane = threadIdx.x % LANES;
  const int which = blockIdx.y;  // 0: keys, 1: values
  __nv_bfloat16* const dst = which ? a.dst[1] : a.dst[0];
  const long long tok = which ? a.tok[1] : a.tok[0], head = which ? a.head[1] : a.head[0];
  void* const pool = which ? a.pool.v : a.pool.k;
  float* const scales = which ? a.pool.v_scale : a.pool.k_scale;
  const long long step = (long long)gridDim.x * (THREADS / LANES);
  for (long long r = (long long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; r < rows; r += step) {
    const long long t = r / a.pool.Hkv;
    const int h = (int)(r - t * a.pool.Hkv);
    const long long slot = slot_of(a.slots, a.wide, t);
    uint4 out = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot < a.pool.pages << a.pool.page_shift) {
      const long long row = pool_row(slot, h, a.pool.Hkv, a.pool.page_shift);
      if constexpr (F == kBf16) {
        out = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(pool) + row * D + lane * 8);
      } else {
        const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + row * D + lane * 8);
        const float scale = scales[row];
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t two = (j < 2 ? q.x : q.y) >> (16 * (j & 1));
          const __nv_bfloat162 p = __floats2bfloat162_rn(__fmul_rn(value_of<F>(two & 0xff), scale),
                                                         __fmul_rn(value_of<F>((two >> 8) & 0xff), scale));
          w[j] = *reinterpret_cast<const uint32_t*>(&p);
        }
        out = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *reinterpret_cast<uint4*>(dst + t * tok + h * head + lane * 8) = out;
  }
}

static dim3 row_grid(long long rows, int D, int sms) {
  const long long per_block = THREADS / (D / 8), blocks = (rows + per_block - 1) / per_block;
  return dim3((unsigned)(blocks < sms * 8ll ? blocks : sms * 8ll), 2);
}

cudaError_t launch_write(const WriteArgs& a, int sms, cudaStream_t stream) {
  const dim3 grid = row_grid(a.T * a.pool.Hkv, a.pool.D, sms);
  by_format(a.pool, [&](auto f, auto d) { write_kernel<decltype(f)::value, decltype(d)::value><<<grid, THREADS, 0, stream>>>(a); });
  return cudaGetLastError();
}

cudaError_t launch_read(const ReadArgs& a, int sms, cudaStream_t stream) {
  const dim3 grid = row_grid(a.T * a.pool.Hkv, a.pool.D, sms);
  by_format(a.pool, [&](auto f, auto d) { read_kernel<decltype(f)::value, decltype(d)::value><<<grid, THREADS, 0, stream>>>(a); });
  return cudaGetLastError();
}

}  // namespace kv
}  // namespace ht
