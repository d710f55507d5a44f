// Arguments and launchers of the text-generation kernels (paged key/value cache, attention over it,
// token sampling).  This header and the kernels' sources use no PyTorch headers; generation.cpp checks
// tensors and fills the arguments in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

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

struct WriteArgs {
  Pool pool;
  const __nv_bfloat16* src[2];  // k, v: [T, Hkv, D]
  long long tok[2], head[2];    // strides in elements
  const void* slots;
  long long T;
  int wide;  // int64 slots
};

struct ReadArgs {
  Pool pool;
  __nv_bfloat16* dst[2];  // [T, Hkv, D]
  long long tok[2], head[2];
  const void* slots;
  long long T;
  int wide;
};

cudaError_t launch_write(const WriteArgs& a, int sms, cudaStream_t stream);
cudaError_t launch_read(const ReadArgs& a, int sms, cudaStream_t stream);

}  // namespace kv

namespace paged {

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
  float* partial;     // workspace_floats(): what a block leaves of a row that other blocks share
  unsigned* arrived;  // workspace_counters(): zero before the first call; every call leaves them zero
};

// Scratch of one call on a GPU with this many SMs.
long long workspace_floats(int sms);
int workspace_counters(int sms);
cudaError_t launch(const Args& a, int sms, cudaStream_t stream);

}  // namespace paged

namespace sampling {

constexpr int kMaxVocabulary = 1 << 18;
constexpr int kMostListed = 2048;  // rows of a batch that the streaming kernel picks its own from

// One value per row, or one for all of them.
template <typename T>
struct PerRow {
  const T* rows;
  T same;
  __host__ __device__ T operator[](int row) const { return rows != nullptr ? rows[row] : same; }
};

struct Args {
  const void* logits;
  long long row_stride, noise_stride;
  const float* noise;
  PerRow<float> temperature, top_p, min_p;
  PerRow<int> top_k;
  long long* token;
  float* logprob;
  int B, V;
  int wide;  // fp32 logits
  float* partial;     // where `streams` says so, workspace_floats(): what a block leaves of a row that other blocks share
  unsigned* arrived;  // likewise workspace_counters(): zero before the first call; every call leaves them zero
  int streamed;       // set by `launch`: rows that the streaming kernel takes are not this launch's
};

// Whether a call takes the kernel for many rows of which nothing is cut (sampling_stream.cu), for all rows (`whole`) or for those
// that turn out to be such, and the scratch that it needs on a GPU with this many SMs.
bool streams(const Args& a, int sms);
long long workspace_floats(int sms);
int workspace_counters(int sms);
cudaError_t launch_stream(const Args& a, bool whole, int sms, cudaStream_t stream);
cudaError_t launch(const Args& a, int sms, cudaStream_t stream);

}  // namespace sampling
}  // namespace ht
