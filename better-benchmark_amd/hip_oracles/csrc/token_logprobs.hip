// Log probabilities of given tokens, with entropy and top alternatives, and
// their gradient.  Per row of logits x, with s_j = scale * x_j:
//   m = max_j s_j,  Z = sum_j e^(s_j - m),  lse = m + ln Z,
//   logprob = (s_t - m) - ln Z,
//   entropy = ln Z - sum_j e^(s_j - m) (s_j - m) / Z,
// and the gradient of  g logprob + g_H entropy + g_lse lse:
//   dx_j = scale * (g [j = t] + p_j (g_lse - g - g_H (ln p_j + H))),
//   p_j = e^(s_j - lse),  p_j ln p_j = 0 where p_j = 0.
//
// The maximum and the two sums are kept while the row streams by (a running
// maximum; the sums are rescaled when it rises), so a row is read once.
// (s_j - m) is formed as scale * (x_j - m): the type's lowest value in every
// place, a row masked by it, then is a row of equal logits and not an
// overflow.
#include <math.h>

#include "hipo_common.h"

namespace hipo {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 64;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();

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

// The running maximum of x with Z = sum 2^u and U = sum 2^u u over
// u = c (x - m), c = scale log2(e).
struct Stats {
  float m, z, u;
};

// u of one value; the clamp keeps 2^u u from being 0 * inf (2^-200 is 0).
__device__ __forceinline__ float exponent(float x, float m, float c) {
  return __builtin_elementwise_maximum((x - m) * c, -200.0f);
}

__device__ __forceinline__ Stats merge(Stats a, Stats b, float c) {
  const float m = __builtin_elementwise_maximum(a.m, b.m);
  // Nothing above -inf on either side, or +inf or NaN on one: finish() needs
  // the maximum alone.
  if (!(fabsf(m) < kInf)) return Stats{m, 0.0f, 0.0f};
  const float ua = exponent(a.m, m, c), ub = exponent(b.m, m, c);
  const float ea = __builtin_amdgcn_exp2f(ua), eb = __builtin_amdgcn_exp2f(ub);
  // sum 2^(u + ua) (u + ua) = 2^ua (U + ua Z)
  return Stats{m, a.z * ea + b.z * eb, ea * (a.u + ua * a.z) + eb * (b.u + ub * b.z)};
}

// What a row's statistics say: its lse and entropy, and s - lse of a value.
struct Row {
  float m, log_z, lse, entropy;
};

__device__ __forceinline__ Row finish(Stats s, float scale) {
  Row r;
  r.m = s.m;
  if (fabsf(s.m) < kInf) {
    r.log_z = kLn2 * __builtin_amdgcn_logf(s.z);
    r.lse = __builtin_fmaf(scale, s.m, r.log_z);
    r.entropy = r.log_z - kLn2 * (s.u / s.z);
  } else {  // -inf: nothing is left; +inf; NaN
    r.log_z = 0.0f;
    r.lse = s.m;
    r.entropy = __builtin_nanf("");
  }
  return r;
}

// In fp64: x - m of the type's lowest and largest value overflows fp32 where
// their scaled difference need not.
__device__ __forceinline__ float log_prob(float x, const Row& r, float scale) {
  const double s = scale;
  return static_cast<float>(fabsf(r.m) < kInf ? s * (double{x} - double{r.m}) - double{r.log_z}
                                              : s * double{x} - double{r.lse});
}

// Order of the alternatives as a whole number: the larger value first (NaN
// above all, -0 with 0), of equal ones the lower index.  0 is no value's.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  uint32_t b = __float_as_uint(x + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (x != x) b = 0xffffffffu;
  return (static_cast<uint64_t>(b) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) {
  return 0xffffffffu - static_cast<uint32_t>(key);
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int size, int64_t i) {
  return size == 8 ? static_cast<const int64_t*>(tokens)[i]
                   : static_cast<const int32_t*>(tokens)[i];
}

struct FwdArgs {
  const void* x;
  const void* tokens;
  float *logprob, *lse, *entropy, *top_logprob;
  int64_t* top_token;
  int64_t rows, vocab, row_stride, ignore_index;
  float scale;
  int token_size, top;
};

// A workgroup per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_rows(FwdArgs a) {
  __shared__ Stats part[kThreads];
  __shared__ uint64_t best[kThreads];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t token = token_at(a.tokens, a.token_size, row);
  if (token == a.ignore_index) {
    if (tid == 0) {
      a.logprob[row] = 0.0f;
      a.lse[row] = 0.0f;
      if (a.entropy) a.entropy[row] = 0.0f;
    }
    for (int i = tid; i < a.top; i += kThreads) {
      a.top_logprob[row * a.top + i] = -kInf;
      a.top_token[row * a.top + i] = -1;
    }
    return;
  }
  const T* x = static_cast<const T*>(a.x) + row * a.row_stride;
  const float c = a.scale * kLog2e;
  Stats s{-kInf, 0.0f, 0.0f};
  for (int64_t j = tid; j < a.vocab; j += kThreads) s = merge(s, Stats{to_f32(x[j]), 1.0f, 0.0f}, c);
  part[tid] = s;
  __syncthreads();
  for (int w = kThreads / 2; w > 0; w /= 2) {
    if (tid < w) part[tid] = merge(part[tid], part[tid + w], c);
    __syncthreads();
  }
  const Row r = finish(part[0], a.scale);
  if (tid == 0) {
    a.logprob[row] = token >= 0 && token < a.vocab ? log_prob(to_f32(x[token]), r, a.scale)
                                                   : __builtin_nanf("");
    a.lse[row] = r.lse;
    if (a.entropy) a.entropy[row] = r.entropy;
  }
  uint64_t last = ~uint64_t{0};
  for (int i = 0; i < a.top; ++i) {
    uint64_t key = 0;
    for (int64_t j = tid; j < a.vocab; j += kThreads) {
      const uint64_t k = order_key(to_f32(x[j]), static_cast<uint32_t>(j));
      if (k < last && k > key) key = k;
    }
    best[tid] = key;
    __syncthreads();
    for (int w = kThreads / 2; w > 0; w /= 2) {
      if (tid < w && best[tid + w] > best[tid]) best[tid] = best[tid + w];
      __syncthreads();
    }
    last = best[0];
    __syncthreads();
    if (tid == 0) {
      const uint32_t j = key_index(last);
      a.top_logprob[row * a.top + i] = log_prob(to_f32(x[j]), r, a.scale);
      a.top_token[row * a.top + i] = j;
    }
  }
}

struct BwdArgs {
  const float* grad;
  const void* x;
  const void* tokens;
  const float *lse, *entropy, *grad_entropy, *grad_lse;
  void* dx;
  int64_t rows, vocab, row_stride, dx_row_stride, ignore_index;
  float scale;
  int token_size;
};

// A workgroup per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_rows(BwdArgs a) {
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.row_stride;
  T* dx = static_cast<T*>(a.dx) + row * a.dx_row_stride;
  const int64_t token = token_at(a.tokens, a.token_size, row);
  if (token == a.ignore_index) {
    for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) dx[j] = from_f32<T>(0.0f);
    return;
  }
  const bool known = token >= 0 && token < a.vocab;
  const float g = known ? a.grad[row] : __builtin_nanf("");
  const float lse = a.lse[row];
  const float gh = a.grad_entropy ? a.grad_entropy[row] : 0.0f;
  const float h = a.grad_entropy ? a.entropy[row] : 0.0f;
  const float factor = (a.grad_lse ? a.grad_lse[row] : 0.0f) - g;
  for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) {
    // The clamp (e^-104 is 0) also keeps p ln p from being 0 * inf.
    const float lp = exp_domain(__builtin_fmaf(a.scale, to_f32(x[j]), -lse));
    float d = exp_f32(lp) * (factor - gh * (lp + h));
    if (j == token) d += g;
    dx[j] = from_f32<T>(a.scale * d);
  }
}

}  // namespace
}  // namespace hipo

extern "C" size_t hipo_token_logprobs_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int hipo_token_logprobs(const void* logits, int elem_size, const void* tokens,
                                   int token_size, float* logprob, float* lse, float* entropy,
                                   float* top_logprob, int64_t* top_token, int64_t rows,
                                   int64_t vocab, int64_t row_stride, float scale,
                                   int64_t ignore_index, int64_t top, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  using namespace hipo;
  clear_error();
  HIPO_REQUIRE(rows >= 0 && vocab >= 0, "token_logprobs: negative size");
  HIPO_REQUIRE(elem_size == 2 || elem_size == 4, "token_logprobs: elem_size must be 2 or 4");
  HIPO_REQUIRE(token_size == 4 || token_size == 8, "token_logprobs: token_size must be 4 or 8");
  HIPO_REQUIRE(scale > 0.0f && scale < __builtin_inff(),
               "token_logprobs: scale must be positive and finite");
  HIPO_REQUIRE(vocab <= 0x7fffffff && rows <= 0x7fffffff, "token_logprobs: size over 2^31");
  HIPO_REQUIRE(row_stride >= vocab, "token_logprobs: row_stride %lld < vocab %lld",
               (long long)row_stride, (long long)vocab);
  HIPO_REQUIRE(top >= 0 && top <= kMaxTop && top <= vocab,
               "token_logprobs: top must be at most %d and at most vocab", kMaxTop);
  if (rows == 0) return 0;
  HIPO_REQUIRE(vocab > 0, "token_logprobs: empty vocabulary");
  HIPO_REQUIRE(logits != nullptr && tokens != nullptr && logprob != nullptr && lse != nullptr,
               "token_logprobs: null pointer");
  HIPO_REQUIRE(top == 0 || (top_logprob != nullptr && top_token != nullptr),
               "token_logprobs: null pointer (top)");
  HIPO_REQUIRE(workspace_bytes >= hipo_token_logprobs_workspace_bytes(rows, vocab, top),
               "token_logprobs: workspace too small");
  const FwdArgs a{logits, tokens, logprob, lse, entropy, top_logprob, top_token, rows, vocab,
                  row_stride, ignore_index, scale, token_size, static_cast<int>(top)};
  auto kernel = elem_size == 2 ? logprobs_rows<uint16_t> : logprobs_rows<float>;
  kernel<<<dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, stream>>>(a);
  return check_launch("token_logprobs");
}

extern "C" int hipo_token_logprobs_bwd(const float* grad, const void* logits, int elem_size,
                                       const void* tokens, int token_size, const float* lse,
                                       const float* entropy, const float* grad_entropy,
                                       const float* grad_lse, void* dlogits, int64_t rows,
                                       int64_t vocab, int64_t row_stride,
                                       int64_t dlogits_row_stride, float scale,
                                       int64_t ignore_index, hipStream_t stream) {
  using namespace hipo;
  clear_error();
  HIPO_REQUIRE(rows >= 0 && vocab >= 0, "token_logprobs_bwd: negative size");
  HIPO_REQUIRE(elem_size == 2 || elem_size == 4, "token_logprobs_bwd: elem_size must be 2 or 4");
  HIPO_REQUIRE(token_size == 4 || token_size == 8,
               "token_logprobs_bwd: token_size must be 4 or 8");
  HIPO_REQUIRE(scale > 0.0f && scale < __builtin_inff(),
               "token_logprobs_bwd: scale must be positive and finite");
  HIPO_REQUIRE(vocab <= 0x7fffffff && rows <= 0x7fffffff, "token_logprobs_bwd: size over 2^31");
  HIPO_REQUIRE(row_stride >= vocab && dlogits_row_stride >= vocab,
               "token_logprobs_bwd: row_stride < vocab %lld", (long long)vocab);
  HIPO_REQUIRE(grad_entropy == nullptr || entropy != nullptr,
               "token_logprobs_bwd: grad_entropy needs the entropy");
  HIPO_REQUIRE(dlogits != logits || dlogits_row_stride == row_stride,
               "token_logprobs_bwd: in place needs one row_stride");
  if (rows == 0 || vocab == 0) return 0;
  HIPO_REQUIRE(grad != nullptr && logits != nullptr && tokens != nullptr && lse != nullptr &&
                   dlogits != nullptr,
               "token_logprobs_bwd: null pointer");
  const BwdArgs a{grad, logits, tokens, lse, entropy, grad_entropy, grad_lse, dlogits, rows,
                  vocab, row_stride, dlogits_row_stride, ignore_index, scale, token_size};
  auto kernel = elem_size == 2 ? logprobs_bwd_rows<uint16_t> : logprobs_bwd_rows<float>;
  kernel<<<dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, stream>>>(a);
  return check_launch("token_logprobs_bwd");
}
