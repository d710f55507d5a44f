// Attention of one new token per sequence over a paged key/value cache.
//
// For query head h of sequence b, with n = lengths[b] tokens in the cache and k_t, v_t the rows of
// its key/value head (times their scales where the pool holds 8 bits):
//     s_t = scale * q . k_t,   o = sum_t softmax(s)_t v_t,   lse = log sum_t exp(s_t).
// A sequence without tokens gives o = 0 and lse = -inf.  Tokens in pages that lie outside the pool
// count as masked, lengths beyond the table are cut to it.
//
// One warp per (sequence, query head), the head's dimensions spread over the lanes, one pass over
// the tokens with the running maximum and sum of the softmax in fp32.
#include "common.cuh"

#include "kv_cache.cuh"

namespace ht {
namespace paged {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Args {
  const __nv_bfloat16* q;  // [B, H, D]
  long long q_seq, q_head;
  kv::Pool pool;
  const int* table;  // [B, width]
  long long table_row;
  int width;
  const int* lengths;
  __nv_bfloat16* out;  // [B, H, D]
  float* lse;          // [B, H] or null
  int B, H;
  float scale_log2;
};

template <int F>
__device__ __forceinline__ float element(const void* pool, long long i) {
  if constexpr (F == kv::kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(pool)[i]);
  if constexpr (F == kv::kInt8) return (float)static_cast<const int8_t*>(pool)[i];
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const __nv_fp8_storage_t*>(pool)[i], __NV_E4M3)));
}

template <int F, int D>
__global__ void __launch_bounds__(128) decode_kernel(Args a) {
  constexpr int E = D / 32;
  const int item = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (item >= a.B * a.H) return;
  const int b = item / a.H, h = item % a.H, g = h / (a.H / a.pool.Hkv);
  const long long n = min((long long)max(a.lengths[b], 0), (long long)a.width << a.pool.page_shift);
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = bf2f(a.q[b * a.q_seq + h * a.q_head + e * 32 + lane]);
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (long long t = 0; t < n; ++t) {
    const int page = a.table[b * a.table_row + (t >> a.pool.page_shift)];
    if (page < 0 || page >= a.pool.pages) continue;
    const long long row = (((long long)page * a.pool.Hkv + g) << a.pool.page_shift) + (t & ((1 << a.pool.page_shift) - 1));
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * element<F>(a.pool.k, row * D + e * 32 + lane);
    s = warp_sum(s) * a.scale_log2 * (F == kv::kBf16 ? 1.f : a.pool.k_scale[row]);
    const float top = fmaxf(m, s);
    const float keep = top == -INFINITY ? 1.f : exp2f(m - top), p = top == -INFINITY ? 0.f : exp2f(s - top);
    const float pv = p * (F == kv::kBf16 ? 1.f : a.pool.v_scale[row]);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * keep + pv * element<F>(a.pool.v, row * D + e * 32 + lane);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) a.out[(long long)item * D + e * 32 + lane] = f2bf(l > 0.f ? o[e] / l : (l == 0.f ? 0.f : l));
  if (lane == 0 && a.lse != nullptr) a.lse[item] = l > 0.f ? m * LN2 + logf(l) : (l == 0.f ? -INFINITY : l);
}

}  // namespace paged

void paged_attention(at::Tensor q, at::Tensor k_pool, at::Tensor v_pool, c10::optional<at::Tensor> k_scale,
                     c10::optional<at::Tensor> v_scale, at::Tensor block_table, at::Tensor lengths, at::Tensor out,
                     c10::optional<at::Tensor> lse, double scale) {
  const c10::cuda::CUDAGuard guard(k_pool.device());
  const kv::Pool p = kv::checked_pool(k_pool, v_pool, k_scale, v_scale);
  HT_CHECK(q.is_cuda() && q.device() == k_pool.device() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == p.D &&
               q.size(1) % p.Hkv == 0 && q.size(1) > 0,
           "q must be a CUDA bf16 tensor [B, H, ", p.D, "] with H a multiple of the pool's ", p.Hkv, " heads");
  const int64_t B = q.size(0), H = q.size(1);
  HT_CHECK(block_table.is_cuda() && block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B &&
               (block_table.size(1) <= 1 || block_table.stride(1) == 1),
           "block_table must be a CUDA int32 tensor [B, pages per sequence] with unit inner stride");
  HT_CHECK(lengths.is_cuda() && lengths.scalar_type() == at::kInt && lengths.is_contiguous() && lengths.dim() == 1 && lengths.size(0) == B,
           "lengths must be a contiguous CUDA int32 tensor [B]");
  HT_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.sizes() == q.sizes(), "out must be contiguous bf16 [B, H, D]");
  if (B == 0) return;
  if (q.stride(2) != 1) q = q.contiguous();
  paged::Args a{reinterpret_cast<const __nv_bfloat16*>(q.data_ptr()), q.stride(0), q.stride(1), p, block_table.data_ptr<int>(),
                block_table.stride(0), (int)block_table.size(1), lengths.data_ptr<int>(),
                reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), nullptr, (int)B, (int)H, (float)(scale * 1.4426950408889634)};
  if (lse.has_value() && lse->defined()) {
    HT_CHECK(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->numel() == B * H, "lse must be contiguous fp32 [B, H]");
    a.lse = lse->data_ptr<float>();
  }
  kv::by_format(p, [&](auto f, auto d) {
    paged::decode_kernel<decltype(f)::value, decltype(d)::value><<<(unsigned)((B * H + 3) / 4), 128, 0, stream()>>>(a);
  });
  HT_CUDA_CHECK(cudaGetLastError());
}

}  // namespace ht
