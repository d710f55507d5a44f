// The paged key/value pool as the kernels that write, read and attend to it see it.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace ht {
namespace kv {

enum Format : int { kBf16 = 0, kInt8 = 1, kFp8 = 2 };

// Smallest scale that a row is stored with (2^-64): its reciprocal is finite, and its logarithm keeps
// the attention kernel's per-token factors inside fp32.
constexpr float kMinScale = 5.421010862427522e-20f;

struct Pool {
  void *k, *v;               // [pages, Hkv, page_size, D]
  float *k_scale, *v_scale;  // [pages, Hkv, page_size] (8-bit formats)
  long long pages;
  int Hkv, page_shift, D, format;
};

inline Pool checked_pool(const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& ks,
                         const c10::optional<at::Tensor>& vs) {
  HT_CHECK(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes() &&
               v.scalar_type() == k.scalar_type() && v.device() == k.device(),
           "key and value pools must be contiguous CUDA tensors [pages, Hkv, page_size, D] of one type");
  const int64_t page = k.size(2);
  HT_CHECK(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page_size must be 16, 32, 64, 128 or 256, got ", page);
  HT_CHECK(k.size(3) == 64 || k.size(3) == 128, "the paged cache supports head_dim 64 or 128, got ", k.size(3));
  HT_CHECK(k.size(0) * page <= INT32_MAX && k.size(1) >= 1 && k.size(1) <= 65535, "the pool holds too many slots or heads");
  int format = kBf16;
  if (k.scalar_type() == at::kChar) format = kInt8;
  else if (k.scalar_type() == at::kFloat8_e4m3fn) format = kFp8;
  else HT_CHECK(k.scalar_type() == at::kBFloat16, "the pool must be bfloat16, int8 or float8_e4m3fn");
  Pool p{k.data_ptr(), v.data_ptr(), nullptr, nullptr, k.size(0), (int)k.size(1), __builtin_ctzll((unsigned long long)page), (int)k.size(3), format};
  if (format != kBf16) {
    HT_CHECK(ks.has_value() && vs.has_value() && ks->defined() && vs->defined(), "an 8-bit pool needs its scales");
    for (const at::Tensor& s : {*ks, *vs})
      HT_CHECK(s.scalar_type() == at::kFloat && s.is_contiguous() && s.device() == k.device() && s.dim() == 3 && s.size(0) == k.size(0) &&
                   s.size(1) == k.size(1) && s.size(2) == page,
               "scales must be contiguous fp32 [pages, Hkv, page_size] on the pool's device");
    p.k_scale = ks->data_ptr<float>();
    p.v_scale = vs->data_ptr<float>();
  }
  HT_CHECK(reinterpret_cast<uintptr_t>(p.k) % 16 == 0 && reinterpret_cast<uintptr_t>(p.v) % 16 == 0, "pools must be 16-byte aligned");
  return p;
}

// Calls launch(format, head size) with both as compile-time constants.
template <typename Launch>
inline void by_format(const Pool& p, const Launch& launch) {
  const auto by_dim = [&](auto format) {
    if (p.D == 128) launch(format, std::integral_constant<int, 128>());
    else launch(format, std::integral_constant<int, 64>());
  };
  if (p.format == kBf16) by_dim(std::integral_constant<int, kBf16>());
  else if (p.format == kInt8) by_dim(std::integral_constant<int, kInt8>());
  else by_dim(std::integral_constant<int, kFp8>());
}

}  // namespace kv
}  // namespace ht
