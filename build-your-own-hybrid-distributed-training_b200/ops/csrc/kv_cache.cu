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
#include "common.cuh"

#include "kv_cache.cuh"

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

struct WriteArgs {
  const __nv_bfloat16* src[2];  // k, v: [T, Hkv, D]
  long long tok[2], head[2];    // strides in elements
  void* dst[2];                 // pools
  float* scale[2];
  const void* slots;
  long long T, capacity;
  int Hkv, page_shift, wide;  // wide: int64 slots
};

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
  const long long rows = a.T * a.Hkv;
  const int lane = threadIdx.x % LANES;
  const int which = blockIdx.y;
  const long long step = (long long)gridDim.x * (THREADS / LANES);
  const long long first = (long long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
  // every lane of a warp makes the same number of turns, so the shuffles below always see a full warp
  for (long long base = first; base - threadIdx.x / LANES < rows; base += step) {
    const bool on = base < rows;
    const long long t = on ? base / a.Hkv : 0;
    const int h = on ? (int)(base - t * a.Hkv) : 0;
    const long long slot = on ? slot_of(a.slots, a.wide, t) : -1;
    const bool stored = slot >= 0 && slot < a.capacity;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (stored) raw = *reinterpret_cast<const uint4*>(a.src[which] + t * a.tok[which] + h * a.head[which] + lane * 8);
    const long long row = stored ? pool_row(slot, h, a.Hkv, a.page_shift) : 0;
    if constexpr (F == kBf16) {
      if (stored) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.dst[which]) + row * D + lane * 8) = raw;
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
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.dst[which]) + row * D + lane * 8) = q;
        if (lane == 0) a.scale[which][row] = scale;
      }
    }
  }
}

struct ReadArgs {
  const void* src[2];
  const float* scale[2];
  __nv_bfloat16* dst[2];  // [T, Hkv, D]
  long long tok[2], head[2];
  const void* slots;
  long long T, capacity;
  int Hkv, page_shift, wide;
};

template <int F, int D>
__global__ void __launch_bounds__(THREADS) read_kernel(ReadArgs a) {
  constexpr int LANES = D / 8;
  const long long rows = a.T * a.Hkv;
  const int lane = threadIdx.x % LANES;
  const int which = blockIdx.y;
  const long long step = (long long)gridDim.x * (THREADS / LANES);
  for (long long r = (long long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; r < rows; r += step) {
    const long long t = r / a.Hkv;
    const int h = (int)(r - t * a.Hkv);
    const long long slot = slot_of(a.slots, a.wide, t);
    uint4 out = make_uint4(0, 0, 0, 0);
    if (slot >= 0 && slot < a.capacity) {
      const long long row = pool_row(slot, h, a.Hkv, a.page_shift);
      if constexpr (F == kBf16) {
        out = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.src[which]) + row * D + lane * 8);
      } else {
        const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.src[which]) + row * D + lane * 8);
        const float scale = a.scale[which][row];
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
    *reinterpret_cast<uint4*>(a.dst[which] + t * a.tok[which] + h * a.head[which] + lane * 8) = out;
  }
}

}  // namespace kv

static void check_rows(const at::Tensor& x, const char* name, int64_t heads, int64_t dim) {
  HT_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() == 3 && x.size(1) == heads && x.size(2) == dim, name,
           " must be a CUDA bf16 tensor [T, ", heads, ", ", dim, "]");
}

static void check_slots(const at::Tensor& slots, const at::Tensor& rows) {
  HT_CHECK(slots.is_cuda() && slots.device() == rows.device() && (slots.scalar_type() == at::kLong || slots.scalar_type() == at::kInt) &&
               slots.dim() == 1 && slots.size(0) == rows.size(0),
           "slots must be an int32 or int64 tensor of one slot per token, on the rows' device");
}

static bool vector_rows(const at::Tensor& x) {
  return x.stride(2) == 1 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}

static dim3 row_grid(long long rows, int D) {
  const int per_block = kv::THREADS / (D / 8);
  return dim3((unsigned)std::max(1ll, std::min((rows + per_block - 1) / per_block, (long long)num_sms() * 8)), 2);
}

void kv_cache_write(at::Tensor k_pool, at::Tensor v_pool, c10::optional<at::Tensor> k_scale, c10::optional<at::Tensor> v_scale,
                    at::Tensor k, at::Tensor v, at::Tensor slots) {
  const c10::cuda::CUDAGuard guard(k_pool.device());
  const kv::Pool p = kv::checked_pool(k_pool, v_pool, k_scale, v_scale);
  check_rows(k, "k", p.Hkv, p.D);
  check_rows(v, "v", p.Hkv, p.D);
  HT_CHECK(k.size(0) == v.size(0) && k.device() == k_pool.device() && v.device() == k_pool.device(),
           "k and v must hold the same tokens, on the pool's device");
  check_slots(slots, k);
  if (k.size(0) == 0) return;
  // rows that a 16-byte load cannot take (another order or alignment) are copied first
  if (!vector_rows(k)) k = k.clone(at::MemoryFormat::Contiguous);
  if (!vector_rows(v)) v = v.clone(at::MemoryFormat::Contiguous);
  slots = slots.contiguous();
  kv::WriteArgs a{{reinterpret_cast<const __nv_bfloat16*>(k.data_ptr()), reinterpret_cast<const __nv_bfloat16*>(v.data_ptr())},
                  {k.stride(0), v.stride(0)},
                  {k.stride(1), v.stride(1)},
                  {p.k, p.v},
                  {p.k_scale, p.v_scale},
                  slots.data_ptr(),
                  k.size(0),
                  (long long)p.pages << p.page_shift,
                  p.Hkv,
                  p.page_shift,
                  slots.scalar_type() == at::kLong};
  const dim3 grid = row_grid(a.T * a.Hkv, p.D);
  kv::by_format(p, [&](auto f, auto d) { kv::write_kernel<decltype(f)::value, decltype(d)::value><<<grid, kv::THREADS, 0, stream()>>>(a); });
  HT_CUDA_CHECK(cudaGetLastError());
}

void kv_cache_read(at::Tensor k_pool, at::Tensor v_pool, c10::optional<at::Tensor> k_scale, c10::optional<at::Tensor> v_scale,
                   at::Tensor slots, at::Tensor k, at::Tensor v) {
  const c10::cuda::CUDAGuard guard(k_pool.device());
  const kv::Pool p = kv::checked_pool(k_pool, v_pool, k_scale, v_scale);
  check_rows(k, "k", p.Hkv, p.D);
  check_rows(v, "v", p.Hkv, p.D);
  HT_CHECK(k.size(0) == v.size(0) && k.device() == k_pool.device() && v.device() == k_pool.device(),
           "k and v must hold the same tokens, on the pool's device");
  check_slots(slots, k);
  if (k.size(0) == 0) return;
  HT_CHECK(vector_rows(k) && vector_rows(v), "k and v must have unit inner stride and rows on 16-byte boundaries");
  slots = slots.contiguous();
  kv::ReadArgs a{{p.k, p.v},
                 {p.k_scale, p.v_scale},
                 {reinterpret_cast<__nv_bfloat16*>(k.data_ptr()), reinterpret_cast<__nv_bfloat16*>(v.data_ptr())},
                 {k.stride(0), v.stride(0)},
                 {k.stride(1), v.stride(1)},
                 slots.data_ptr(),
                 k.size(0),
                 (long long)p.pages << p.page_shift,
                 p.Hkv,
                 p.page_shift,
                 slots.scalar_type() == at::kLong};
  const dim3 grid = row_grid(a.T * a.Hkv, p.D);
  kv::by_format(p, [&](auto f, auto d) { kv::read_kernel<decltype(f)::value, decltype(d)::value><<<grid, kv::THREADS, 0, stream()>>>(a); });
  HT_CUDA_CHECK(cudaGetLastError());
}

}  // namespace ht
