// Entry points of the text-generation kernels: checks of the tensors, scratch memory, launches.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <utility>

#include "generation.cuh"

namespace ht {
namespace {

#define HT_CHECK(cond, ...) TORCH_CHECK(cond, __VA_ARGS__)

void check_launch(cudaError_t err, const char* what) {
  TORCH_CHECK(err == cudaSuccess, "CUDA error: ", cudaGetErrorString(err), " in ", what);
}

int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

kv::Pool checked_pool(const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& ks, const c10::optional<at::Tensor>& vs) {
  HT_CHECK(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes() &&
               v.scalar_type() == k.scalar_type() && v.device() == k.device(),
           "key and value pools must be contiguous CUDA tensors [pages, Hkv, page_size, D] of one type");
  const int64_t page = k.size(2);
  HT_CHECK(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page_size must be 16, 32, 64, 128 or 256, got ", page);
  HT_CHECK(k.size(3) == 64 || k.size(3) == 128, "the paged cache supports head_dim 64 or 128, got ", k.size(3));
  HT_CHECK(k.size(0) * page <= INT32_MAX && k.size(1) >= 1 && k.size(1) <= 65535, "the pool holds too many slots or heads");
  int format = kv::kBf16;
  if (k.scalar_type() == at::kChar) format = kv::kInt8;
  else if (k.scalar_type() == at::kFloat8_e4m3fn) format = kv::kFp8;
  else HT_CHECK(k.scalar_type() == at::kBFloat16, "the pool must be bfloat16, int8 or float8_e4m3fn");
  kv::Pool p{k.data_ptr(), v.data_ptr(), nullptr, nullptr, k.size(0), (int)k.size(1), __builtin_ctzll((unsigned long long)page),
             (int)k.size(3), format};
  if (format != kv::kBf16) {
    HT_CHECK(ks.has_value() && vs.has_value() && ks->defined() && vs->defined(), "an 8-bit pool needs its scales");
    for (const at::Tensor* s : {&*ks, &*vs})
      HT_CHECK(s->scalar_type() == at::kFloat && s->is_contiguous() && s->device() == k.device() && s->dim() == 3 && s->size(0) == k.size(0) &&
                   s->size(1) == k.size(1) && s->size(2) == page && reinterpret_cast<uintptr_t>(s->data_ptr()) % 16 == 0,
               "scales must be contiguous, 16-byte aligned fp32 [pages, Hkv, page_size] on the pool's device");
    p.k_scale = ks->data_ptr<float>();
    p.v_scale = vs->data_ptr<float>();
  }
  HT_CHECK(reinterpret_cast<uintptr_t>(p.k) % 16 == 0 && reinterpret_cast<uintptr_t>(p.v) % 16 == 0, "pools must be 16-byte aligned");
  return p;
}

void check_rows(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots, const at::Tensor& pool) {
  for (const at::Tensor* x : {&k, &v})
    HT_CHECK(x->device() == pool.device() && x->scalar_type() == at::kBFloat16 && x->dim() == 3 && x->size(0) == k.size(0) &&
                 x->size(1) == pool.size(1) && x->size(2) == pool.size(3),
             "k and v must be bf16 [T, ", pool.size(1), ", ", pool.size(3), "] on the pool's device");
  HT_CHECK(slots.device() == pool.device() && (slots.scalar_type() == at::kLong || slots.scalar_type() == at::kInt) && slots.dim() == 1 &&
               slots.size(0) == k.size(0),
           "slots must be int32 or int64, one per token, on the pool's device");
  HT_CHECK(k.size(0) <= (1ll << 30) / pool.size(1), "too many rows (tokens x heads) for one call: split it");
}

void check_no_gradient(const at::Tensor& x, const char* what) {
  HT_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()), what, " has no gradient: call it under torch.no_grad()");
}

// Rows that 16-byte accesses can take.
bool vector_rows(const at::Tensor& x) {
  return x.stride(2) == 1 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}

// Scratch of the kernels that join what several blocks leave of a row.  Calls on one stream follow one another, so they share
// one buffer per (device, stream); a captured call gets memory of its own graph, since replays may run on any stream.
std::pair<float*, unsigned*> join_scratch(const at::Tensor& like, cudaStream_t stream, at::Tensor& keep) {
  const long long floats = std::max(paged::workspace_floats(sms()), sampling::workspace_floats(sms()));
  const long long bytes = floats * 4 + std::max(paged::workspace_counters(sms()), sampling::workspace_counters(sms())) * 4;
  const auto split = [&](const at::Tensor& t) {
    char* base = static_cast<char*>(t.data_ptr());
    return std::make_pair(reinterpret_cast<float*>(base), reinterpret_cast<unsigned*>(base + floats * 4));
  };
  const auto fresh = [&] {
    at::Tensor t = at::empty({bytes}, like.options().dtype(at::kByte));
    check_launch(cudaMemsetAsync(static_cast<char*>(t.data_ptr()) + floats * 4, 0, bytes - floats * 4, stream), "scratch");
    return t;
  };
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  check_launch(cudaStreamIsCapturing(stream, &status), "cudaStreamIsCapturing");
  if (status != cudaStreamCaptureStatusNone) {
    keep = fresh();
    return split(keep);
  }
  // never destroyed: at exit the CUDA context may be gone before static objects are
  static auto* mutex = new std::mutex;
  static auto* buffers = new std::map<std::pair<int, cudaStream_t>, at::Tensor>;
  const std::lock_guard<std::mutex> lock(*mutex);
  at::Tensor& t = (*buffers)[{like.get_device(), stream}];
  if (!t.defined()) t = fresh();
  return split(t);
}

template <typename T>
sampling::PerRow<T> per_row(const c10::optional<at::Tensor>& t, double same, const at::Tensor& logits, at::ScalarType type, const char* name) {
  if (!t.has_value() || !t->defined()) return {nullptr, (T)same};
  HT_CHECK(t->device() == logits.device() && t->scalar_type() == type && t->is_contiguous() && t->dim() == 1 && t->size(0) == logits.size(0),
           name, " must be a number or a contiguous ", type, " tensor [B] on the logits' device");
  return {t->data_ptr<T>(), (T)same};
}

}  // namespace

void kv_cache_write(at::Tensor k_pool, at::Tensor v_pool, c10::optional<at::Tensor> k_scale, c10::optional<at::Tensor> v_scale,
                    at::Tensor k, at::Tensor v, at::Tensor slots) {
  const kv::Pool p = checked_pool(k_pool, v_pool, k_scale, v_scale);
  check_rows(k, v, slots, k_pool);
  check_no_gradient(k, "kv_cache_write");
  check_no_gradient(v, "kv_cache_write");
  if (k.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(k_pool.device());
  // rows of another order or alignment are copied first
  if (!vector_rows(k)) k = k.clone(at::MemoryFormat::Contiguous);
  if (!vector_rows(v)) v = v.clone(at::MemoryFormat::Contiguous);
  if (slots.size(0) > 1) slots = slots.contiguous();
  const kv::WriteArgs a{p,
                        {reinterpret_cast<const __nv_bfloat16*>(k.data_ptr()), reinterpret_cast<const __nv_bfloat16*>(v.data_ptr())},
                        {k.stride(0), v.stride(0)},
                        {k.stride(1), v.stride(1)},
                        slots.data_ptr(),
                        k.size(0),
                        slots.scalar_type() == at::kLong};
  check_launch(kv::launch_write(a, sms(), at::cuda::getCurrentCUDAStream()), "kv_cache_write");
}

std::tuple<at::Tensor, at::Tensor> kv_cache_read(at::Tensor k_pool, at::Tensor v_pool, c10::optional<at::Tensor> k_scale,
                                                 c10::optional<at::Tensor> v_scale, at::Tensor slots, c10::optional<at::Tensor> k_out,
                                                 c10::optional<at::Tensor> v_out) {
  const kv::Pool p = checked_pool(k_pool, v_pool, k_scale, v_scale);
  const c10::cuda::CUDAGuard guard(k_pool.device());
  HT_CHECK(slots.dim() == 1 && k_out.has_value() == v_out.has_value(), "slots must be a vector, and out a pair");
  const auto fresh = [&] { return at::empty({slots.size(0), p.Hkv, p.D}, k_pool.options().dtype(at::kBFloat16)); };
  at::Tensor k = k_out.has_value() ? *k_out : fresh(), v = v_out.has_value() ? *v_out : fresh();
  check_rows(k, v, slots, k_pool);
  if (k.size(0) == 0) return {k, v};
  HT_CHECK(vector_rows(k) && vector_rows(v), "k and v must have unit inner stride and rows on 16-byte boundaries");
  if (slots.size(0) > 1) slots = slots.contiguous();
  const kv::ReadArgs a{p,
                       {reinterpret_cast<__nv_bfloat16*>(k.data_ptr()), reinterpret_cast<__nv_bfloat16*>(v.data_ptr())},
                       {k.stride(0), v.stride(0)},
                       {k.stride(1), v.stride(1)},
                       slots.data_ptr(),
                       k.size(0),
                       slots.scalar_type() == at::kLong};
  check_launch(kv::launch_read(a, sms(), at::cuda::getCurrentCUDAStream()), "kv_cache_read");
  return {k, v};
}

std::tuple<at::Tensor, c10::optional<at::Tensor>> paged_attention(at::Tensor q, at::Tensor k_pool, at::Tensor v_pool,
                                                                  c10::optional<at::Tensor> k_scale, c10::optional<at::Tensor> v_scale,
                                                                  at::Tensor block_table, at::Tensor lengths, c10::optional<double> scale,
                                                                  bool with_lse) {
  const kv::Pool p = checked_pool(k_pool, v_pool, k_scale, v_scale);
  check_no_gradient(q, "paged_attention");
  HT_CHECK(q.device() == k_pool.device() && q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == p.D &&
               q.size(1) % p.Hkv == 0 && q.size(1) > 0 && q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX,
           "q must be bf16 [B, H, ", p.D, "] on the pool's device with H a multiple of the pool's ", p.Hkv, " heads");
  const int64_t B = q.size(0), H = q.size(1);
  HT_CHECK(block_table.device() == q.device() && block_table.scalar_type() == at::kInt && block_table.dim() == 2 &&
               block_table.size(0) == B && (block_table.size(1) <= 1 || block_table.stride(1) == 1) && block_table.size(1) * k_pool.size(2) <= INT32_MAX - 256,
           "block_table must be int32 [B, pages per sequence] with unit inner stride, on the pool's device");
  HT_CHECK(B * ((block_table.size(1) * k_pool.size(2) + 15) / 16) < (1ll << 31) / H,
           "block_table spans too many tokens for one call (sequences x heads x tokens / 16 beyond 2^31): split the batch");
  HT_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kInt && lengths.is_contiguous() && lengths.dim() == 1 &&
               lengths.size(0) == B,
           "lengths must be a contiguous int32 tensor [B] on the pool's device");
  const c10::cuda::CUDAGuard guard(k_pool.device());
  at::Tensor out = at::empty({B, H, p.D}, q.options().requires_grad(false));
  c10::optional<at::Tensor> lse;
  if (with_lse) lse = at::empty({B, H}, q.options().dtype(at::kFloat).requires_grad(false));
  if (B == 0) return {out, lse};
  if (!vector_rows(q)) q = q.clone(at::MemoryFormat::Contiguous);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  paged::Args a{reinterpret_cast<const __nv_bfloat16*>(q.data_ptr()), q.stride(0), q.stride(1), p, block_table.data_ptr<int>(),
                block_table.stride(0), (int)block_table.size(1), lengths.data_ptr<int>(),
                reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), with_lse ? lse->data_ptr<float>() : nullptr, (int)B, (int)H,
                (float)((scale.has_value() ? *scale : 1.0 / std::sqrt((double)p.D)) * 1.4426950408889634), nullptr, nullptr};
  at::Tensor keep;
  std::tie(a.partial, a.arrived) = join_scratch(q, stream, keep);
  check_launch(paged::launch(a, sms(), stream), "paged_attention");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> sample_tokens(at::Tensor logits, at::Tensor noise, c10::optional<at::Tensor> temperature_rows,
                                                 double temperature, c10::optional<at::Tensor> top_k_rows, int64_t top_k,
                                                 c10::optional<at::Tensor> top_p_rows, double top_p,
                                                 c10::optional<at::Tensor> min_p_rows, double min_p) {
  HT_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
           "logits must be a CUDA bf16 or fp32 tensor [B, V]");
  const int64_t B = logits.size(0), V = logits.size(1);
  HT_CHECK(V >= 1 && V <= sampling::kMaxVocabulary && B <= (1 << 24), "sample_tokens supports 1 to ", sampling::kMaxVocabulary,
           " tokens and up to 2^24 rows, got ", V, " and ", B);
  HT_CHECK(noise.device() == logits.device() && noise.scalar_type() == at::kFloat && noise.sizes() == logits.sizes(),
           "noise must be an fp32 tensor of the logits' shape and device");
  const auto in_range = [](double x, double most) { return x >= 0.0 && x <= most; };  // false for NaN
  HT_CHECK(in_range(temperature, INFINITY) && top_k >= 0 && in_range(top_p, 1.0) && in_range(min_p, 1.0),
           "temperature and top_k must be 0 or more, top_p and min_p between 0 and 1");
  check_no_gradient(logits, "sample_tokens");
  const c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor token = at::empty({B}, logits.options().dtype(at::kLong).requires_grad(false));
  at::Tensor logprob = at::empty({B}, logits.options().dtype(at::kFloat).requires_grad(false));
  if (B == 0) return {token, logprob};
  if (V > 1 && logits.stride(1) != 1) logits = logits.contiguous();
  if (V > 1 && noise.stride(1) != 1) noise = noise.contiguous();
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  sampling::Args a{logits.data_ptr(),
                   logits.stride(0),
                   noise.stride(0),
                   noise.data_ptr<float>(),
                   per_row<float>(temperature_rows, temperature, logits, at::kFloat, "temperature"),
                   per_row<float>(top_p_rows, top_p, logits, at::kFloat, "top_p"),
                   per_row<float>(min_p_rows, min_p, logits, at::kFloat, "min_p"),
                   per_row<int>(top_k_rows, (double)std::min<int64_t>(top_k, V), logits, at::kInt, "top_k"),
                   reinterpret_cast<long long*>(token.data_ptr<int64_t>()),
                   logprob.data_ptr<float>(),
                   (int)B,
                   (int)V,
                   logits.scalar_type() == at::kFloat,
                   nullptr,
                   nullptr,
                   0};
  at::Tensor keep;
  if (sampling::streams(a, sms())) std::tie(a.partial, a.arrived) = join_scratch(logits, stream, keep);
  check_launch(sampling::launch(a, sms(), stream), "sample_tokens");
  return {token, logprob};
}

}  // namespace ht
