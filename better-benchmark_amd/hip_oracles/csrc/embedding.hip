// Embedding lookup with a scale, and its gradient:
//   out[t] = scale * w[token_t],    dw[v] = scale * sum_{t: token_t = v} grad[t],
// the sum in fp32 in an order that the shape alone fixes, one rounding at the
// end.
#include <math.h>

#include "hipo_common.h"

namespace hipo {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<uint16_t>(uint16_t v) {
  return bf16_to_f32(v);
}
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ uint16_t from_f32<uint16_t>(float v) {
  return static_cast<uint16_t>(pack_bf16x2(v, 0.0f) & 0xffffu);
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int size, int64_t i) {
  return size == 8 ? static_cast<const int64_t*>(tokens)[i]
                   : static_cast<const int32_t*>(tokens)[i];
}

struct FwdArgs {
  const void* w;
  const void* tokens;
  void* out;
  int64_t count, width, vocab, row_stride;
  float scale;
  int token_size;
};

// A workgroup per token.
template <typename T>
__global__ __launch_bounds__(kThreads) void embedding_rows(FwdArgs a) {
  const int64_t t = blockIdx.x;
  const int64_t v = token_at(a.tokens, a.token_size, t);
  const bool known = v >= 0 && v < a.vocab;
  const T* w = static_cast<const T*>(a.w) + (known ? v : 0) * a.row_stride;
  T* out = static_cast<T*>(a.out) + t * a.width;
  for (int64_t j = threadIdx.x; j < a.width; j += kThreads)
    out[j] = from_f32<T>(known ? to_f32(w[j]) * a.scale : __builtin_nanf(""));
}

struct BwdArgs {
  const void* grad;
  const void* tokens;
  void* dw;
  int64_t count, width, vocab, padding_idx;
  float scale;
  int token_size, accumulate;
};

// A workgroup per row of dw, which looks for its tokens.
template <typename T, typename O>
__global__ __launch_bounds__(kThreads) void embedding_bwd_rows(BwdArgs a) {
  __shared__ int found[kThreads];
  __shared__ int count;
  const int64_t v = blockIdx.x;
  const int tid = threadIdx.x;
  const T* grad = static_cast<const T*>(a.grad);
  O* dw = static_cast<O*>(a.dw) + v * a.width;
  bool any = false;
  for (int64_t j0 = 0; j0 < a.width; j0 += kThreads) {
    const int64_t j = j0 + tid;
    float sum = 0.0f;
    any = false;
    for (int64_t t0 = 0; t0 < a.count; t0 += kThreads) {
      const int64_t t = t0 + tid;
      found[tid] = t < a.count && v != a.padding_idx && token_at(a.tokens, a.token_size, t) == v;
      if (tid == 0) count = 0;
      __syncthreads();
      if (found[tid]) count = 1;
      __syncthreads();
      if (count) {
        any = true;
        for (int i = 0; i < kThreads; ++i)
          if (found[i] && j < a.width) sum += to_f32(grad[(t0 + i) * a.width + j]);
      }
      __syncthreads();
    }
    if (j < a.width) {
      if (!a.accumulate) {
        dw[j] = from_f32<O>(sum * a.scale);
      } else if (any) {
        dw[j] = from_f32<O>(to_f32(dw[j]) + sum * a.scale);
      }
    }
  }
}

}  // namespace
}  // namespace hipo

extern "C" int hipo_embedding(const void* weight, int elem_size, const void* tokens,
                              int token_size, void* out, int64_t count, int64_t width,
                              int64_t vocab, int64_t row_stride, float scale,
                              hipStream_t stream) {
  using namespace hipo;
  clear_error();
  HIPO_REQUIRE(count >= 0 && width >= 0 && vocab >= 0, "embedding: negative size");
  HIPO_REQUIRE(elem_size == 2 || elem_size == 4, "embedding: elem_size must be 2 or 4");
  HIPO_REQUIRE(token_size == 4 || token_size == 8, "embedding: token_size must be 4 or 8");
  HIPO_REQUIRE(count <= 0x7fffffff && width <= 0x7fffffff && vocab <= 0x7fffffff,
               "embedding: size over 2^31");
  HIPO_REQUIRE(row_stride >= width, "embedding: row_stride %lld < width %lld",
               (long long)row_stride, (long long)width);
  if (count == 0 || width == 0) return 0;
  HIPO_REQUIRE(vocab > 0, "embedding: empty vocabulary");
  HIPO_REQUIRE(weight != nullptr && tokens != nullptr && out != nullptr,
               "embedding: null pointer");
  const FwdArgs a{weight, tokens, out, count, width, vocab, row_stride, scale, token_size};
  auto kernel = elem_size == 2 ? embedding_rows<uint16_t> : embedding_rows<float>;
  kernel<<<dim3(static_cast<unsigned>(count)), dim3(kThreads), 0, stream>>>(a);
  return check_launch("embedding");
}

extern "C" size_t hipo_embedding_bwd_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int hipo_embedding_bwd(const void* grad, int elem_size, const void* tokens,
                                  int token_size, void* dweight, int out_size, int64_t count,
                                  int64_t width, int64_t vocab, float scale,
                                  int64_t padding_idx, int accumulate, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  using namespace hipo;
  clear_error();
  HIPO_REQUIRE(count >= 0 && width >= 0 && vocab >= 0, "embedding_bwd: negative size");
  HIPO_REQUIRE((elem_size == 2 || elem_size == 4) && (out_size == 2 || out_size == 4),
               "embedding_bwd: elem_size and out_size must be 2 or 4");
  HIPO_REQUIRE(token_size == 4 || token_size == 8, "embedding_bwd: token_size must be 4 or 8");
  HIPO_REQUIRE(count <= 0x7fffffff && width <= 0x7fffffff && vocab <= 0x7fffffff,
               "embedding_bwd: size over 2^31");
  if (width == 0 || vocab == 0) return 0;
  HIPO_REQUIRE(dweight != nullptr && (count == 0 || (grad != nullptr && tokens != nullptr)),
               "embedding_bwd: null pointer");
  HIPO_REQUIRE(workspace_bytes >= hipo_embedding_bwd_workspace_bytes(count, width, vocab),
               "embedding_bwd: workspace too small");
  const BwdArgs a{grad, tokens, dweight, count, width, vocab, padding_idx, scale, token_size,
                  accumulate};
  auto kernel = elem_size == 2 ? (out_size == 2 ? embedding_bwd_rows<uint16_t, uint16_t>
                                                : embedding_bwd_rows<uint16_t, float>)
                               : (out_size == 2 ? embedding_bwd_rows<float, uint16_t>
                                                : embedding_bwd_rows<float, float>);
  kernel<<<dim3(static_cast<unsigned>(vocab)), dim3(kThreads), 0, stream>>>(a);
  return check_launch("embedding_bwd");
}
