// Log probabilities of given tokens, with entropy and top alternatives, and
// their gradient.  Per row of logits x, with s_j = scale * x_j:
//   m = max_j s_j,  Z = sum_j e^(s_j - m),  lse = m + ln Z,
//   logprob = (s_t - m) - ln Z,
//   entropy = ln Z - sum_j e^(s_j - m) (s_j - m) / Z,
// and the gradient of  g logprob + g_H entropy + g_lse lse:
//   dx_j = scale * (g [j = t] + p_j (g_lse - g - g_H (ln p_j + H))),
//   p_j = e^(s_j - lse),  p_j ln p_j = 0 where p_j = 0.
//
// Forward: HBM-bound, the row is read once.  Each lane keeps a running
// maximum and the two sums relative to it (rescaled when it rises, at most once
// per round of 8 to 64 values); lanes, waves and slices of a row are then joined
// by the same rescaling, so that a row's bits depend on its values, on where in 16
// bytes it begins and on the plan, on no other row.  A workgroup takes a row, or a
// slice of one where there are too few rows to fill the chip, whose parts a second
// launch joins.
//
// For the alternatives nothing is kept while the row streams by: the lanes' maxima
// say where the largest values are.  The k-th largest of 64 groups' maxima is
// a lower bound of the k-th largest value, few values reach it (k = 20: about
// 24), and they lie in lanes whose maximum does: only these lanes' values are
// read again, shared out over the workgroup, and ranked by counting.  With 0 / 20 /
// 33 / 64 alternatives, us, bf16: [1, 32000] 5.6 / 8.7 / 9.0 / 12.8, [64, 128000] 9.2 /
// 13.6 / 15.3 / 57, [4096, 16384] 25 / 38 / 45 / 140.  Rows of one value cost a
// second search for its first places (20 alternatives: 28, 42, 165).  Where more
// than 1024 values lie above all but a few lanes' they are found one by one, a pass
// over the row or slice each (every second run of 32 vectors far above the others:
// 33 alternatives 160, 269, 1256; 64 alternatives 286, 491, 2295).
//
// Backward: HBM-bound, one pass, a value's gradient needs its logit and a few
// numbers of its row.
#include <math.h>

#include <algorithm>

#include "hipo_common.h"

namespace hipo {
namespace {

constexpr int kThreads = 256;
constexpr int kLarge = 1024;       // threads of a workgroup where rows are few
constexpr int kMaxTop = 64;
constexpr int64_t kMaxSlices = 64;    // of a row
constexpr int kCandidates = 1024;  // values that a slice can rank at once
constexpr int64_t kMaxVocab = 0x7fffffff - 4096;
constexpr int64_t kMaxBlocks = 1 << 23;  // of a launch
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();
constexpr float kFar = 0x1p20f;

// C consecutive logits in 16 bytes.
template <typename T>
struct Logits {
  static constexpr int C = 16 / sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(C)));
  typedef Vec Unaligned __attribute__((aligned(sizeof(T))));
};

__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }

__device__ __forceinline__ void unpack(u32x4_t v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16lo(v[i]);
    x[2 * i + 1] = bf16hi(v[i]);
  }
}
__device__ __forceinline__ void unpack(u32x4_t v, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
}

__device__ __forceinline__ u32x4_t pack(const float (&x)[8]) {
  return u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                 pack_bf16x2(x[6], x[7])};
}
__device__ __forceinline__ u32x4_t pack(const float (&x)[4]) {
  return u32x4_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                 __float_as_uint(x[3])};
}

__device__ __forceinline__ float maximum(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

__device__ __forceinline__ int64_t token_at(const void* tokens, int size, int64_t i) {
  return size == 8 ? static_cast<const int64_t*>(tokens)[i]
                   : static_cast<const int32_t*>(tokens)[i];
}

// ---------------------------------------------------------------------------
// Statistics: the maximum m of x, Z = sum 2^w and U = sum 2^w w, where w is
// c x less a reference near c m, c = scale log2(e).  Near (c m below 2^20) the
// reference is c m rounded, and w one FMA per value: exact before its one
// rounding, and 2^-5 off c (x - m) at most, which finish() puts back.  Far (a
// row of nothing but mask values of -1e9, or of the type's lowest) it is c m
// itself and w = c (x - m): the rounding of c m could be any number there.
// m = -inf: nothing yet.
// ---------------------------------------------------------------------------

struct Stats {
  float m, z, u;
};

// -round(c m); 0 for -inf, so that w of -inf is -inf.
__device__ __forceinline__ float offset(float m, float c) { return m == -kInf ? 0.0f : -(m * c); }

__device__ __forceinline__ bool is_far(float o) { return !(fabsf(o) < kFar); }  // NaN too

// 2^w w without 0 * inf (2^-200 is 0).
__device__ __forceinline__ float weighted(float e, float w) { return e * maximum(w, -200.0f); }

// s relative to the maximum m >= s.m instead.
__device__ __forceinline__ Stats rescale(Stats s, float m, float c) {
  if (s.m == m) return s;
  const float o = offset(m, c), had = offset(s.m, c);
  // The old reference less the new one, in one rounding each.
  float d = o - had;
  if (__builtin_expect(is_far(o) || is_far(had), 0)) {
    d = !is_far(o)    ? __builtin_fmaf(s.m, c, o)
        : is_far(had) ? (s.m - m) * c
                      : __builtin_fmaf(-m, c, -had);
  }
  // s.m = -inf: its sums are 0, and 2^d is at most 1 (a NaN m stays in m).
  d = __builtin_elementwise_minimum(maximum(d, -200.0f), 0.0f);
  const float f = __builtin_amdgcn_exp2f(d);
  return Stats{m, s.z * f, f * __builtin_fmaf(d, s.z, s.u)};
}

template <int N, bool ENTROPY>
__device__ __forceinline__ void add_values(Stats& s, const float (&x)[N], float c) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) top = maximum(maximum(top, x[i]), x[i + 1]);
  if constexpr (N % 2 == 0) top = maximum(top, x[N - 1]);
  const float m = maximum(s.m, top);
  s = rescale(s, m, c);
  const float o = offset(m, c);
  float z[2] = {0.0f, 0.0f}, u[2] = {0.0f, 0.0f};
  if (__builtin_expect(is_far(o), 0)) {
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      float v = x[0];  // x[i], kept in registers
#pragma unroll
      for (int k = 1; k < N; ++k) v = i == k ? x[k] : v;
      const float w = maximum((v - m) * c, -200.0f);
      const float e = __builtin_amdgcn_exp2f(w);
      z[0] += e;
      u[0] += e * w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float w = __builtin_fmaf(x[i], c, o);
      const float e = __builtin_amdgcn_exp2f(w);
      z[i & 1] += e;
      if constexpr (ENTROPY) u[i & 1] += weighted(e, w);
    }
  }
  s.z += z[0] + z[1];
  if constexpr (ENTROPY) s.u += u[0] + u[1];
}

// Of all lanes of a wave, and of a workgroup's waves; every lane has it.
__device__ __forceinline__ Stats join_wave(Stats s, float c) {
  const float m = wave_maximum(s.m);
  s = rescale(s, m, c);
  return Stats{m, wave_sum(s.z), wave_sum(s.u)};
}

// Of n <= 64 parts, a part per lane; every lane has it.
__device__ __forceinline__ Stats join_parts(const Stats* part, int n, float c) {
  const int lane = threadIdx.x & (kWave - 1);
  return join_wave(lane < n ? part[lane] : Stats{-kInf, 0.0f, 0.0f}, c);
}

struct Row {
  float m, log_z, lse, entropy;
};

// Z and U relative to m itself.  The largest value's own term is e_m = 2^(w of
// m), the same bits here as in Z, and sums of positive terms never fall below
// one of them: Z / e_m >= 1, and exactly 1 where one value is all there is.  So
// ln Z >= 0: no log probability is above 0, no entropy below.
__device__ __forceinline__ Row finish(Stats s, float scale, float c) {
  // U - w_m Z, two roundings of one product: 0 where one value is all there is.
#pragma clang fp contract(off)
  Row r;
  r.m = s.m;
  if (fabsf(s.m) < kInf) {
    const float o = offset(s.m, c);
    const float w_m = is_far(o) ? 0.0f : __builtin_fmaf(s.m, c, o);
    r.log_z = maximum(kLn2 * __builtin_amdgcn_logf(s.z / __builtin_amdgcn_exp2f(w_m)), 0.0f);
    r.lse = __builtin_fmaf(scale, s.m, r.log_z);
    r.entropy = maximum(r.log_z + kLn2 * ((w_m * s.z - s.u) / s.z), 0.0f);
  } else {  // -inf: nothing is left; +inf; NaN
    r.log_z = 0.0f;
    r.lse = s.m;
    r.entropy = __builtin_nanf("");
  }
  return r;
}

// s - lse of a value.  In fp64: x - m of the type's lowest and largest value
// overflows fp32 where their scaled difference need not.
__device__ __forceinline__ float log_prob(float x, const Row& r, float scale) {
  const double s = scale;
  return static_cast<float>(fabsf(r.m) < kInf ? s * (double{x} - double{r.m}) - double{r.log_z}
                                              : s * double{x} - double{r.lse});
}

// ---------------------------------------------------------------------------
// Order of the alternatives as whole numbers: the larger value first (NaN
// above all, -0 with 0), of equal ones the lower index.  0 is no value's.
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0xffffffffu ? __builtin_nanf("")
                          : __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t order_key(uint32_t order, uint32_t index) {
  return (static_cast<uint64_t>(order) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_order(uint64_t key) {
  return static_cast<uint32_t>(key >> 32);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) {
  return 0xffffffffu - static_cast<uint32_t>(key);
}

// The k-th largest of a wave's 64 orders (0 if fewer than k are not 0), bit by
// bit the largest number that k of them reach; with 16 BITS its upper ones,
// a lower bound (bf16 values have no others).
template <int BITS>
__device__ __forceinline__ uint32_t kth_of_wave(uint32_t order, int k) {
  uint32_t v = 0;
#pragma unroll
  for (int b = 31; b >= 32 - BITS; --b) {
    const uint32_t higher = v | (1u << b);
    if (__popcll(__ballot(order >= higher)) >= k) v = higher;
  }
  return v;
}

// Writes the k largest of n keys in falling order to sorted (all of a
// workgroup's threads; keys are distinct, n >= k).
template <int NT>
__device__ __forceinline__ void sort_top(const uint64_t* keys, int n, int k, uint64_t* sorted) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t key = keys[i];
    int above = 0;
#pragma unroll 8
    for (int l = 0; l < n; ++l) above += keys[l] > key ? 1 : 0;
    if (above < k) sorted[above] = key;
  }
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------

struct FwdArgs {
  const void* x;
  const void* tokens;
  float *logprob, *lse, *entropy, *top_logprob;
  int64_t* top_token;
  Stats* parts;      // [rows][slices]
  uint64_t* keys;    // [rows][slices][kMaxTop]
  int64_t first, vocab, row_stride, ignore_index;
  float scale, c;
  int token_size, top, slices, span;  // of span 16-byte vectors
  int rounds;                         // vectors per lane in a slice
  DivMagic by_slices, by_rounds;
};

template <int NT>
__device__ __forceinline__ void write_ignored(const FwdArgs& a, int64_t row) {
  if (threadIdx.x == 0) {
    a.logprob[row] = 0.0f;
    a.lse[row] = 0.0f;
    if (a.entropy) a.entropy[row] = 0.0f;
  }
  for (int i = threadIdx.x; i < a.top; i += NT) {
    a.top_logprob[row * a.top + i] = -kInf;
    a.top_token[row * a.top + i] = -1;
  }
}

template <int NT>
__device__ __forceinline__ void write_row(const FwdArgs& a, int64_t row, int64_t token, float at,
                                          const Row& r, const uint64_t* sorted) {
  if (threadIdx.x == 0) {
    a.logprob[row] =
        token >= 0 && token < a.vocab ? log_prob(at, r, a.scale) : __builtin_nanf("");
    a.lse[row] = r.lse;
    if (a.entropy) a.entropy[row] = r.entropy;
  }
  for (int i = threadIdx.x; i < a.top; i += NT) {
    const uint64_t key = sorted[i];
    a.top_logprob[row * a.top + i] = log_prob(value_of(key_order(key)), r, a.scale);
    a.top_token[row * a.top + i] = key_index(key);
  }
}

// A slice of a row: 16-byte vectors lo..hi of those that are aligned in
// memory, and for the row's first slice the values before the first and after
// the last of them, one per lane.
template <typename T>
struct Slice {
  const T* x;      // the row
  const T* vec;    // its first aligned vector
  int head;        // values before it
  int lo, hi;
  int odd;         // this lane's odd value's index, -1: none

  static constexpr int C = Logits<T>::C;

  __device__ __forceinline__ Slice(const FwdArgs& a, int64_t row, int slice) {
    x = static_cast<const T*>(a.x) + row * a.row_stride;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const int vocab = static_cast<int>(a.vocab);
    head = std::min(off == 0 ? 0 : C - off, vocab);
    vec = x + head;
    const int n = (vocab - head) / C;
    lo = std::min(n, slice * a.span);
    hi = slice == a.slices - 1 ? n : std::min(n, lo + a.span);
    const int tail = vocab - head - n * C;
    const int tid = threadIdx.x;
    odd = slice != 0 || tid >= head + tail ? -1 : tid < head ? tid : vocab - tail + tid - head;
  }
  __device__ __forceinline__ u32x4_t load(int v) const {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(vec) + v);
  }
  __device__ __forceinline__ int index(int v) const { return head + v * C; }
};

template <int NT>
struct TopMemory {
  uint64_t keys[kCandidates + kMaxTop];
  uint64_t sorted[kMaxTop];
  uint32_t lane_order[NT];
  int lanes[NT];  // those whose maximum reaches the bound
  int lane_count, count;
  int wave_count[NT / kWave];
};

// Collects the values of a slice whose order is at least (STRICT: above) tau
// into mem.keys; returns how many there are (which may be more than it holds).
// All threads; lane_order: the order of the thread's maximum.
template <bool STRICT, int NT, typename T>
__device__ __forceinline__ int collect(const Slice<T>& s, DivMagic by_rounds, int rounds,
                                       uint32_t lane_order, uint32_t tau, TopMemory<NT>& mem) {
  constexpr int C = Logits<T>::C;
  constexpr int kLoads = 4;
  // Not below the bound as a value: the same (a NaN bound, of an order below
  // that of -inf or a NaN's, leaves nothing out).
  const float bound = value_of(tau);
  const auto reaches = [&](float v) { return STRICT ? order_of(v) > tau : !(v < bound); };
  if (threadIdx.x == 0) mem.lane_count = mem.count = 0;
  __syncthreads();
  if (lane_order != 0 && (STRICT ? lane_order > tau : lane_order >= tau))
    mem.lanes[atomicAdd(&mem.lane_count, 1)] = threadIdx.x;
  if (s.odd >= 0) {
    const float x = to_f32(s.x[s.odd]);
    if (reaches(x)) {
      const int at = atomicAdd(&mem.count, 1);
      if (at < kCandidates) mem.keys[at] = order_key(order_of(x), static_cast<uint32_t>(s.odd));
    }
  }
  __syncthreads();
  // Their vectors, NT apart, shared out over all threads.
  const int n = mem.lane_count * rounds;
  for (int j0 = threadIdx.x; j0 < n; j0 += NT * kLoads) {
    int v[kLoads];
    u32x4_t raw[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int j = j0 + k * NT;
      v[k] = s.hi;
      if (j < n) {
        const int l = static_cast<int>(div_by(j, by_rounds));
        v[k] = s.lo + (j - l * rounds) * NT + mem.lanes[l];
      }
      if (v[k] < s.hi) raw[k] = s.load(v[k]);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      if (v[k] >= s.hi) continue;
      float x[C];
      unpack(raw[k], x);
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < C; ++i) hits |= reaches(x[i]) ? 1u << i : 0u;
      if (hits == 0) continue;
      int at = atomicAdd(&mem.count, __popc(hits));
      for (; hits != 0; hits &= hits - 1, ++at) {
        const int i = __builtin_ctz(hits);
        float y = x[0];  // x[i], kept in registers
#pragma unroll
        for (int c = 1; c < C; ++c) y = i == c ? x[c] : y;
        if (at < kCandidates)
          mem.keys[at] = order_key(order_of(y), static_cast<uint32_t>(s.index(v[k]) + i));
      }
    }
  }
  __syncthreads();
  return mem.count;
}

// Appends the `want` lowest indexes of values whose order is tau to keys.
template <int NT, typename T>
__device__ __forceinline__ void collect_equal(const Slice<T>& s, uint32_t tau, int want,
                                              uint64_t* keys, int* wave_count) {
  constexpr int C = Logits<T>::C;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  int have = 0;
  // One value per thread, in order of the index: before the vectors, they,
  // and after them.
  const auto step = [&](bool equal, int index) {
    const uint64_t m = __ballot(equal);
    __syncthreads();
    if (lane == 0) wave_count[wave] = __popcll(m);
    __syncthreads();
    int at = have + __popcll(m & ((uint64_t{1} << lane) - 1));
    for (int w = 0; w < NT / kWave; ++w) {
      if (w < wave) at += wave_count[w];
      have += wave_count[w];
    }
    if (equal && at < want) keys[at] = order_key(tau, static_cast<uint32_t>(index));
  };
  const auto is = [&](int index) { return order_of(to_f32(s.x[index])) == tau; };
  step(s.odd >= 0 && s.odd < s.head && is(s.odd), s.odd);
  for (int i = s.lo * C; i < s.hi * C && have < want; i += NT) {
    const int at = i + static_cast<int>(threadIdx.x);
    step(at < s.hi * C && is(s.head + at), s.head + at);
  }
  step(s.odd >= s.head && s.odd >= 0 && is(s.odd), s.odd);
  __syncthreads();
}

// The slice's k largest keys: with sort they alone, in falling order, without
// it at most kMaxTop keys with them among them; returns where, and in n how
// many.  All threads; x: the lane's maximum.
template <int NT, typename T>
__device__ __forceinline__ const uint64_t* slice_top(const Slice<T>& s, DivMagic by_rounds,
                                                     int rounds, float x, bool any, int k,
                                                     bool sort, TopMemory<NT>& mem, int& n) {
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const uint32_t mine = any ? order_of(x) : 0;
  mem.lane_order[tid] = mine;
  if (tid < kMaxTop) mem.sorted[tid] = 0;
  __syncthreads();
  uint32_t group = mem.lane_order[lane];
#pragma unroll
  for (int w = 1; w < NT / kWave; ++w) group = std::max(group, mem.lane_order[w * kWave + lane]);
  uint32_t tau = kth_of_wave<16>(group, k);
  n = collect<false, NT>(s, by_rounds, rounds, mine, tau, mem);
  if (!sort && n <= kMaxTop) return mem.keys;
  if (n > kCandidates) {
    // Many values are equal to the bound, or near it: those above the exact one,
    // and the first of those equal to it.
    tau = kth_of_wave<32>(group, k);
    __syncthreads();
    n = collect<true, NT>(s, by_rounds, rounds, mine, tau, mem);
    if (n < k) {
      collect_equal<NT>(s, tau, k - n, mem.keys + n, mem.wave_count);
      n = k;
    }
  }
  if (n <= kCandidates) {
    sort_top<NT>(mem.keys, n, k, mem.sorted);
    __syncthreads();
    n = std::min(n, k);
    return mem.sorted;
  }
  // Still too many, all in a few lanes: one by one.
  uint64_t last = ~uint64_t{0};
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    const auto look = [&](float v, int index) {
      const uint64_t key = order_key(order_of(v), static_cast<uint32_t>(index));
      // (A NaN at index 0 has the largest key there is.)
      if ((i == 0 || key < last) && key > best) best = key;
    };
    if (s.odd >= 0) look(to_f32(s.x[s.odd]), s.odd);
    for (int v = s.lo + tid; v < s.hi; v += NT) {
      float y[Logits<T>::C];
      unpack(s.load(v), y);
#pragma unroll
      for (int e = 0; e < Logits<T>::C; ++e) look(y[e], s.index(v) + e);
    }
    mem.keys[tid] = best;
    __syncthreads();
    for (int w = NT / 2; w > 0; w /= 2) {
      if (tid < w) mem.keys[tid] = std::max(mem.keys[tid], mem.keys[tid + w]);
      __syncthreads();
    }
    last = mem.keys[0];
    if (tid == 0) mem.sorted[i] = last;
    __syncthreads();
  }
  n = k;
  return mem.sorted;
}

// A workgroup of NT threads per row and slice, kFlight 16-byte loads per lane
// and round.
template <int NT, int kFlight, typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_slices(FwdArgs a) {
  constexpr int C = Logits<T>::C;
  __shared__ Stats wave_stats[NT / kWave];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & (kWave - 1);
  const uint32_t r = div_by(blockIdx.x, a.by_slices);
  const int slice = static_cast<int>(blockIdx.x - r * a.slices);
  const int64_t row = a.first + r;
  const Slice<T> s(a, row, slice);
  Stats stats{-kInf, 0.0f, 0.0f};
  // The next round's loads before this one's values.  (Two sets of registers
  // instead of the copy, so that no load waits for another, measured the same.)
  constexpr int kRound = NT * kFlight;
  u32x4_t next[kFlight];
  const auto load = [&](int v0) {
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int v = v0 + f * NT + tid;
      next[f] = s.load(v < s.hi ? v : s.hi - 1);
    }
  };
  // The first round beside the token, and for nothing where that is ignored.
  if (s.lo < s.hi) load(s.lo);
  __builtin_amdgcn_sched_barrier(0);
  const int64_t token = token_at(a.tokens, a.token_size, row);
  if (token == a.ignore_index) {
    if (a.slices == 1) write_ignored<NT>(a, row);
    return;
  }
  float at = 0.0f;
  if (tid == 0 && a.slices == 1 && token >= 0 && token < a.vocab) at = to_f32(s.x[token]);
  float odd[1] = {-kInf};
  if (s.odd >= 0) odd[0] = to_f32(s.x[s.odd]);
  for (int v0 = s.lo; v0 < s.hi; v0 += kRound) {
    u32x4_t now[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) now[f] = next[f];
    if (v0 + kRound < s.hi) load(v0 + kRound);
    __builtin_amdgcn_sched_barrier(0);
    float x[kFlight * C];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      float y[C];
      unpack(now[f], y);
#pragma unroll
      for (int i = 0; i < C; ++i) x[f * C + i] = y[i];
    }
    if (v0 + kRound > s.hi) {
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        if (v0 + f * NT + tid >= s.hi) {
#pragma unroll
          for (int i = 0; i < C; ++i) x[f * C + i] = -kInf;
        }
      }
    }
    add_values<kFlight * C, ENTROPY>(stats, x, a.c);
  }
  const float lane_max = stats.m;  // of its vectors
  if (slice == 0 && wave == 0) add_values<1, ENTROPY>(stats, odd, a.c);

  const Stats w = join_wave(stats, a.c);
  if (lane == 0) wave_stats[wave] = w;
  __syncthreads();
  const Stats all = NT == kWave ? w : join_parts(wave_stats, NT / kWave, a.c);

  const uint64_t* best = nullptr;
  int n = 0;
  if constexpr (TOP) {
    __shared__ TopMemory<NT> mem;
    // A lane with an odd value alone takes part with it.
    const bool vectors = s.lo + tid < s.hi;
    const float m = s.odd >= 0 ? (vectors ? maximum(lane_max, odd[0]) : odd[0]) : lane_max;
    best = slice_top(s, a.by_rounds, a.rounds, m, vectors || s.odd >= 0, a.top, a.slices == 1, mem,
                     n);
  }
  if (a.slices == 1) {
    write_row<NT>(a, row, token, at, finish(all, a.scale, a.c), best);
    return;
  }
  const int64_t part = row * a.slices + slice;
  if (tid == 0) a.parts[part] = all;
  if constexpr (TOP) {
    // 0 where there is none.
    if (tid < kMaxTop) a.keys[part * kMaxTop + tid] = tid < n ? best[tid] : 0;
  }
}

// Joins the slices of a row: a workgroup per row.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void join_slices(FwdArgs a) {
  constexpr int NT = kThreads;
  __shared__ Stats parts[kMaxSlices];
  const int tid = threadIdx.x;
  const int64_t row = a.first + blockIdx.x;
  const int64_t token = token_at(a.tokens, a.token_size, row);
  if (token == a.ignore_index) {
    write_ignored<NT>(a, row);
    return;
  }
  float at = 0.0f;
  if (tid == 0 && token >= 0 && token < a.vocab)
    at = to_f32(static_cast<const T*>(a.x)[row * a.row_stride + token]);
  if (tid < a.slices) parts[tid] = a.parts[row * a.slices + tid];
  const uint64_t* best = nullptr;
  if constexpr (TOP) {
    // Of the slices' keys those that reach the k-th largest of 64 groups'
    // maxima, sorted.
    __shared__ uint64_t keys[kMaxSlices * kMaxTop];
    __shared__ uint64_t few[kMaxSlices * kMaxTop];
    __shared__ uint64_t sorted[kMaxTop];
    __shared__ int count;
    const int n = a.slices * kMaxTop;
    for (int i = tid; i < n; i += NT) keys[i] = a.keys[row * n + i];
    if (tid == 0) count = 0;
    if (tid < kMaxTop) sorted[tid] = 0;
    __syncthreads();
    uint32_t group = 0;
    // (A slice's first places are the filled ones: another lane's in each.)
    for (int i = 0; i < a.slices; ++i)
      group = std::max(group, key_order(keys[i * kMaxTop + ((tid + 23 * i) & (kMaxTop - 1))]));
    const uint32_t tau = kth_of_wave<16>(group, a.top);
    for (int i = tid; i < n; i += NT) {
      if (keys[i] != 0 && key_order(keys[i]) >= tau) few[atomicAdd(&count, 1)] = keys[i];
    }
    __syncthreads();
    sort_top<NT>(few, count, a.top, sorted);
    best = sorted;
  }
  __syncthreads();
  write_row<NT>(a, row, token, at, finish(join_parts(parts, a.slices, a.c), a.scale, a.c), best);
}

// Threads per workgroup, slices per row and 16-byte vectors per slice, us of
// graph replays on one card (bf16; 0 / 20 alternatives):
//   one wave per row where rows are short and many: [8192, 1000] 8.6 at 64
//   threads, 24.4 at 256; [8192, 8192] 25.4, 25.2; fewer rows only up to 2048
//   values, for the search that one wave does alone ([512, 8192] 6.2 / 13.6 at
//   64, 5.5 / 8.6 at 256).  What is asked for does not enter: the statistics
//   are the same bits with and without alternatives;
//   1024 threads for up to a row per CU where 256 take four rounds of loads or
//   more (256 / 1024 threads, with 20 alternatives: rows of 2900 vectors, three
//   rounds, [1] 7.7 / 8.3, [64] 8.4 / 9.2, [256] 9.8 / 10.4; of 3400, four, [1] 8.3 /
//   8.1, [64] 9.3 / 9.1, [256] 10.5 / 10.4, fp32 9.8 / 9.3; of 8192, [256] 15.1 /
//   12.4; without alternatives 3400 [1] 5.3 / 5.1, [256] 6.7 / 7.1, fp32 6.2 / 6.0.
//   Just past a round of 1024 they lose: 4600 [256] 7.3 / 9.3, 11.7 / 12.5, fp32 7.1 /
//   7.5, 10.9 / 10.8).  [512, 32000] 9.7 / 19.1 at 1024, 9.5 / 13.6 at 256;
//   slices of 16 KB and more of still longer rows where that fills the chip
//   no more than twice: [64, 128000] one slice of 1024 threads 11.9 / 15.8, 4
//   slices 8.9 / 13.7, 8 slices 8.5 / 12.9, 16 slices 8.6 / 14.5; [1, 200000]
//   16.6 / 19.5, 8 slices 7.3 / 11.5, 16 slices 6.1 / 11.0; [256, 128000] 15.6 /
//   19.3, 2 slices 16.5 / 23.6.
//   Loads in flight: 2 per lane where a wave has a row ([16384, 1000] 10.2,
//   with 4 12.6), 8 for many rows of bf16 (2 / 4 / 8: [8192, 50001] - / 136 / 130,
//   [8192, 32000] - / 86 / 81; [512, 32000] 13.8 / 13.4 / 13.5 with 20
//   alternatives, [700, 32000] - / 16.2 / 17.2; fp32 the same either way).
struct Plan {
  int threads, slices, span, flight;
};

inline Plan plan(int64_t rows, int64_t vocab, int elem_size) {
  const int64_t vectors = vocab / (16 / elem_size);
  int64_t slices = 1;
  Plan p;
  if (vectors <= (rows >= 1024 ? 1024 : 256)) {
    p.threads = kWave;
  } else if (rows <= 128 && vectors >= 6144) {
    p.threads = kThreads;
    slices = std::min({std::max<int64_t>(4, 512 / rows), vectors / 1024, kMaxSlices});
  } else {
    const int64_t round = kThreads * 4;
    p.threads = rows <= 256 && (vectors + round - 1) / round >= 4 ? kLarge : kThreads;
  }
  p.flight = rows >= 2048 && elem_size == 2 ? 8 : 4;
  p.span = static_cast<int>(
      ((vectors + slices - 1) / slices + p.threads - 1) / p.threads * p.threads);
  p.slices = slices == 1 ? 1 : static_cast<int>((vectors + p.span - 1) / p.span);
  return p;
}

inline size_t parts_bytes(int64_t rows, int slices) {
  return (rows * slices * sizeof(Stats) + 15) / 16 * 16;
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------

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

// 16-byte vectors per lane, 8 values: us at 1 / 2 / 4 vectors, [8192, 128000]
// bf16 635 / 667 / 728, [1501, 50001] fp32 101 / 95 / 102.
template <typename T>
constexpr int kBwdVectors = 8 / Logits<T>::C;
// Rows per grid layer.  The last layer's workgroups past the rows end at once: just
// past 49152 rows nearly half of all.
constexpr int kBwdRows = 49152;
constexpr int kBwdLineFrom = 1024;  // vectors of a row from which on lines count

// The gradient of a logit, without the token's own term.  e^-104 is 0: the
// bound keeps p ln p from being 0 * inf.
template <bool ENTROPY>
__device__ __forceinline__ float logit_grad(float x, float scale, float lse, float factor,
                                            float gh, float h) {
  const float lp = maximum(__builtin_fmaf(scale, x, -lse), -104.0f);
  const float p = exp_f32(lp);
  return p * (ENTROPY ? factor - gh * (lp + h) : factor);
}

// A workgroup per row and chunk of it: blockIdx.x the chunk, y and z the row.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_chunks(BwdArgs a) {
  constexpr int C = Logits<T>::C, N = kBwdVectors<T>;
  typedef typename Logits<T>::Unaligned Unaligned;
  const int64_t row = static_cast<int64_t>(blockIdx.z) * kBwdRows + blockIdx.y;
  if (row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.row_stride;
  T* dx = static_cast<T*>(a.dx) + row * a.dx_row_stride;
  const int vocab = static_cast<int>(a.vocab);
  // Vectors are aligned in dx.
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(dx) % 16 / sizeof(T));
  const int head = std::min(off == 0 ? 0 : C - off, vocab);
  const int n = (vocab - head) / C;
  const int tail = vocab - head - n * C;
  const int tid = threadIdx.x;
  int odd = -1;
  if (blockIdx.x == 0 && tid < head + tail) odd = tid < head ? tid : vocab - tail + tid - head;
  // Waves of long rows begin on whole 128-byte lines of dx ([4096, 50001] bf16
  // 129.2 -> 127.4 us, [1501, 50001] fp32 97.7 -> 95.2; [16384, 1000] would
  // take 16.9 instead of 15.0).
  const int nt = static_cast<int>(blockDim.x);
  const int line =
      n < kBwdLineFrom ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(dx + head) / 16 % 8);
  const int v0 = static_cast<int>(blockIdx.x) * (nt * N) + tid - line;

  const int64_t token = token_at(a.tokens, a.token_size, row);
  if (token == a.ignore_index) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int v = v0 + k * nt;
      if (v >= 0 && v < n)
        __builtin_nontemporal_store(u32x4_t{0u, 0u, 0u, 0u},
                                    reinterpret_cast<u32x4_t*>(dx + head) + v);
    }
    if (odd >= 0) dx[odd] = T{0};
    return;
  }
  u32x4_t in[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int v = v0 + k * nt;
    if (v >= 0 && v < n)
      in[k] = __builtin_bit_cast(
          u32x4_t,
          __builtin_nontemporal_load(reinterpret_cast<const Unaligned*>(x + head + v * C)));
  }
  const bool known = token >= 0 && token < a.vocab;
  const float g = known ? a.grad[row] : __builtin_nanf("");
  const float lse = a.lse[row];
  const float gh = ENTROPY ? a.grad_entropy[row] : 0.0f;
  const float h = ENTROPY ? a.entropy[row] : 0.0f;
  const float factor = (a.grad_lse ? a.grad_lse[row] : 0.0f) - g;
  const int hot = known ? static_cast<int>(token) : -1;
  const auto gradient = [&](float v, int index) {
    const float d = logit_grad<ENTROPY>(v, a.scale, lse, factor, gh, h);
    return a.scale * (index == hot ? d + g : d);
  };
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int v = v0 + k * nt;
    if (v < 0 || v >= n) continue;
    float f[C];
    unpack(in[k], f);
#pragma unroll
    for (int i = 0; i < C; ++i) f[i] = gradient(f[i], head + v * C + i);
    __builtin_nontemporal_store(pack(f), reinterpret_cast<u32x4_t*>(dx + head) + v);
  }
  if (odd >= 0) {
    const float d = gradient(to_f32(x[odd]), odd);
    if constexpr (sizeof(T) == 2) dx[odd] = static_cast<T>(pack_bf16x2(d, 0.0f) & 0xffffu);
    else dx[odd] = d;
  }
}

}  // namespace
}  // namespace hipo

extern "C" size_t hipo_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
  using namespace hipo;
  if (rows <= 0 || vocab <= 0 || top < 0 || rows > 0x7fffffff || vocab > 0x7fffffff) return 0;
  // The most of either element size.
  const int slices = std::max(plan(rows, vocab, 2).slices, plan(rows, vocab, 4).slices);
  if (slices == 1) return 0;
  return parts_bytes(rows, slices) + (top ? rows * slices * kMaxTop * sizeof(uint64_t) : 0);
}

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
  HIPO_REQUIRE(scale >= 0x1p-100f && scale <= 0x1p100f,
               "token_logprobs: scale must be from 2^-100 to 2^100");
  HIPO_REQUIRE(vocab <= kMaxVocab && rows <= 0x7fffffff,
               "token_logprobs: vocab over 2^31 - 4096 or rows over 2^31");
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
  const size_t need = hipo_token_logprobs_workspace_bytes(rows, vocab, top);
  HIPO_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need),
               "token_logprobs: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  HIPO_REQUIRE(need == 0 || aligned16(workspace),
               "token_logprobs: workspace must be 16-byte aligned");
  const Plan p = plan(rows, vocab, elem_size);
  FwdArgs a{logits, tokens, logprob, lse, entropy, top_logprob, top_token,
                  static_cast<Stats*>(workspace),
                  reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) +
                                              parts_bytes(rows, p.slices)),
                  0, vocab, row_stride, ignore_index, scale, scale * kLog2eHi, token_size,
                  static_cast<int>(top), p.slices, p.span,
                  std::max(1, p.span / p.threads), div_magic(static_cast<uint32_t>(p.slices)),
                  div_magic(static_cast<uint32_t>(std::max(1, p.span / p.threads)))};
  const bool bf16 = elem_size == 2, ent = entropy != nullptr;
#define HIPO_LP(N_, F_, T_)                                   \
  (top ? (ent ? logprobs_slices<N_, F_, T_, true, true>       \
              : logprobs_slices<N_, F_, T_, false, true>)     \
       : (ent ? logprobs_slices<N_, F_, T_, true, false>      \
              : logprobs_slices<N_, F_, T_, false, false>))
#define HIPO_LP_N(N_, F_) (bf16 ? HIPO_LP(N_, F_, uint16_t) : HIPO_LP(N_, F_, float))
  auto kernel = p.threads == kWave    ? HIPO_LP_N(kWave, 2)
                : p.threads == kLarge ? HIPO_LP_N(kLarge, 4)
                : p.flight == 8       ? HIPO_LP(kThreads, 8, uint16_t)
                                      : HIPO_LP_N(kThreads, 4);
#undef HIPO_LP_N
#undef HIPO_LP
  auto join = bf16 ? (top ? join_slices<uint16_t, true> : join_slices<uint16_t, false>)
                   : (top ? join_slices<float, true> : join_slices<float, false>);
  const int64_t step = kMaxBlocks / p.slices;
  for (; a.first < rows; a.first += step) {
    const unsigned n = static_cast<unsigned>(std::min(step, rows - a.first));
    kernel<<<dim3(n * p.slices), dim3(p.threads), 0, stream>>>(a);
    if (p.slices == 1) continue;
    if (const int rc = check_launch("token_logprobs")) return rc;  // nothing to join
    join<<<dim3(n), dim3(kThreads), 0, stream>>>(a);
  }
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
  HIPO_REQUIRE(scale >= 0x1p-100f && scale <= 0x1p100f,
               "token_logprobs_bwd: scale must be from 2^-100 to 2^100");
  HIPO_REQUIRE(vocab <= kMaxVocab && rows <= 0x7fffffff,
               "token_logprobs_bwd: vocab over 2^31 - 4096 or rows over 2^31");
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
  // One vector more, and where lines count one line, than the row is long.  A
  // row's workgroups are alike, so that no half empty one ends it ([15320, 2945]
  // bf16 37.1 us instead of 44.6, [8192, 4097] 25.2 instead of 27.6).
  const int64_t c = 16 / elem_size, per_lane = 8 / c;
  const int64_t vectors = vocab / c + (vocab / c < kBwdLineFrom ? 1 : 9);
  const int64_t lanes = (vectors + per_lane - 1) / per_lane;
  const int64_t groups = (lanes + kThreads - 1) / kThreads;
  const unsigned threads = static_cast<unsigned>(
      ((lanes + groups - 1) / groups + kWave - 1) / kWave * kWave);
  const dim3 grid(static_cast<unsigned>((lanes + threads - 1) / threads),
                  static_cast<unsigned>(std::min<int64_t>(rows, kBwdRows)),
                  static_cast<unsigned>((rows + kBwdRows - 1) / kBwdRows));
  const bool ent = grad_entropy != nullptr;
  auto kernel = elem_size == 2 ? (ent ? logprobs_bwd_chunks<uint16_t, true>
                                      : logprobs_bwd_chunks<uint16_t, false>)
                               : (ent ? logprobs_bwd_chunks<float, true>
                                      : logprobs_bwd_chunks<float, false>);
  kernel<<<grid, dim3(threads), 0, stream>>>(a);
  return check_launch("token_logprobs_bwd");
}
