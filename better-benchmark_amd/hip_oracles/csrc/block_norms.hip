// The norms around a block of a residual network, fused with its gate and the
// residual sum, and their gradient.
//
// With norm(v; w, b) = (v - m) r (offset + w) + b, where r = 1 / sqrt(mean((v -
// m)^2) + eps) and m is the row's mean (LayerNorm) or 0 (RMSNorm):
//   n = norm(x; post),  h = residual + scale gate n,  y = norm(h; pre)
// and backwards, T being the gradient of h from both of its uses:
//   with u = grad_y (offset + pre), e = (h - m) r:
//   T = grad_h + r (u - e mean(u e) - mean(u))        (mean(u): LayerNorm only)
//   dresidual = T,  dpre = sum grad_y e,  dpre_bias = sum grad_y
//   v = scale gate T,  dgate = scale sum T n,  dpost = sum v f,
//   dpost_bias = sum v,  with f the normalised x;  dx as T's second term, of v.
//
// Both passes read every value once and hold the row in registers between its
// statistics and its results; HBM bounds them.  A row belongs to a team of
// lanes with groups of 8 values (16-byte accesses of bf16, 1 KiB of a row per
// wave): up to 512 columns 1 to 64 lanes of one wave with one group each, above
// that whole waves, forwards with two groups a lane, backwards with one up to
// 4096 columns (bwd_groups()).
#include <algorithm>

#include "hipo_common.h"

namespace hipo {
namespace {

constexpr int kGroup = 8;        // values per lane and step
constexpr int kSmallCols = 512;  // one wave or less per row
constexpr int64_t kMostCols = 16384;

struct Vec8 {
  float v[kGroup];
};

// 8 values as they lie in memory, at any element alignment.
template <typename T>
struct Raw8;

template <>
struct Raw8<uint16_t> {
  u32x4_t w;
  __device__ __forceinline__ void load(const uint16_t* p) {
    w = *reinterpret_cast<const u32x4_a2_t*>(p);
  }
  __device__ __forceinline__ void load_once(const uint16_t* p) {
    w = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2_t*>(p));
  }
  __device__ __forceinline__ void clear_unless(bool keep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = keep ? w[i] : 0u;
  }
  __device__ __forceinline__ Vec8 values() const {
    Vec8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.v[2 * i] = bf16lo(w[i]);
      r.v[2 * i + 1] = bf16hi(w[i]);
    }
    return r;
  }
};

template <>
struct Raw8<float> {
  f32x4_t a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4_a4_t*>(p);
    b = *reinterpret_cast<const f32x4_a4_t*>(p + 4);
  }
  __device__ __forceinline__ void load_once(const float* p) { load(p); }
  __device__ __forceinline__ void clear_unless(bool keep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = keep ? a[i] : 0.0f;
      b[i] = keep ? b[i] : 0.0f;
    }
  }
  __device__ __forceinline__ Vec8 values() const {
    return Vec8{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
};

// What every row reads again, and what is read once: bf16 without a place in the
// caches ([8192, 4096], other rows each time: forward 54.1 -> 51.2 us, and 48.9
// with such stores too; gradient 89.5 -> 76.2, with such stores 83.7).  fp32 takes
// two loads a lane, each of half the bytes of a line, and the second would find
// the line gone (gradient of [8192, 4096] 167 -> 210 us).
template <typename T>
__device__ __forceinline__ Vec8 load8(const T* p) {
  Raw8<T> r;
  r.load(p);
  return r.values();
}
template <typename T>
__device__ __forceinline__ Vec8 load8_once(const T* p) {
  Raw8<T> r;
  r.load_once(p);
  return r.values();
}

template <bool Once = false>
__device__ __forceinline__ void store8(uint16_t* p, const Vec8& r) {
  u32x4_t w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(r.v[2 * i], r.v[2 * i + 1]);
  if (Once) {
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4_a2_t*>(p));
  } else {
    *reinterpret_cast<u32x4_a2_t*>(p) = w;
  }
}

template <bool Once = false>
__device__ __forceinline__ void store8(float* p, const Vec8& r) {
  *reinterpret_cast<f32x4_a4_t*>(p) = f32x4_t{r.v[0], r.v[1], r.v[2], r.v[3]};
  *reinterpret_cast<f32x4_a4_t*>(p + 4) = f32x4_t{r.v[4], r.v[5], r.v[6], r.v[7]};
}

__device__ __forceinline__ float as_stored(float v, const uint16_t*) { return round_bf16(v); }
__device__ __forceinline__ float as_stored(float v, const float*) { return v; }

__device__ __forceinline__ void store1(uint16_t* p, float v) {
  *p = static_cast<uint16_t>(pack_bf16x2(v, 0.0f));
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }

// How a launch is cut: teams of `lanes` lanes, `teams` of them in a workgroup.
struct Layout {
  int lanes;  // a power of two up to 64, or a multiple of 64
  int teams;
  int threads() const { return lanes * teams; }
};

// `groups`: of 8 values per lane, where a row has whole waves.
inline Layout layout_of(int64_t cols, int groups) {
  const int64_t pieces = (cols + kGroup - 1) / kGroup;
  if (cols <= kSmallCols) {
    int lanes = 1;
    while (lanes < pieces) lanes *= 2;
    return Layout{lanes, 512 / lanes};
  }
  const int waves = static_cast<int>((pieces + kWave * groups - 1) / (kWave * groups));
  return Layout{waves * kWave, std::max(1, 8 / waves)};
}

// Groups per lane of the gradient: it holds up to nine rows' worth of registers
// (four operands, the next row's, up to five sums), and with one group 8 to 16
// waves fit a CU.  Rows past 4096 columns take two, so that 8 waves hold a row
// and each lane has 256 registers; past 8192 columns 16 waves do, of 128.
inline int bwd_groups(int64_t cols) { return cols <= 512 * kGroup ? 1 : 2; }

// Where a lane's groups lie.  The group that would cross the row's end is moved
// back to end there; its first `skip` values belong to the group before, which
// computes the same bits, and count in no sum.  skip = 8: past the row, owns
// nothing (and loads what the last group loads).
template <int U>
struct Columns {
  int col[U];
  int skip[U];
};

template <int U>
__device__ __forceinline__ Columns<U> columns_of(int place, int lanes, int cols) {
  Columns<U> c;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int first = (u * lanes + place) * kGroup;
    c.col[u] = min(first, cols - kGroup);
    c.skip[u] = min(first - c.col[u], kGroup);
  }
  return c;
}

// Sums over a team, N at once, every lane receiving them, in an order that the
// layout fixes.  `slot`: LDS of N floats per wave, other than the last call's.
template <int N, bool SMALL, int M>
__device__ __forceinline__ void team_sum(float (&v)[M], int lanes, float* slot) {
  if (SMALL) {
    for (int o = 1; o < lanes; o *= 2) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  const int waves = lanes / kWave;
  if (waves == 1) return;
  const int wave = threadIdx.x / kWave;
  if (lane_id() == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slot[wave * N + i] = v[i];
  }
  __syncthreads();
  const float* mine = slot + wave / waves * waves * N;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
  for (int w = 0; w < waves; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += mine[w * N + i];
  }
}

// s[0] += sum w e and, LAYER, s[1] += sum w over the columns a lane owns.
template <int U, bool LAYER>
__device__ __forceinline__ void pair_sum(float (&s)[2], const Vec8 (&w)[U], const Vec8 (&e)[U],
                                         const Columns<U>& c, bool ragged) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float t[2] = {0.0f, 0.0f};
    if (ragged) {  // some lane owns a part of its group
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const float v = i >= c.skip[u] ? w[u].v[i] : 0.0f;
        t[0] += v * (i >= c.skip[u] ? e[u].v[i] : 0.0f);
        if (LAYER) t[1] += v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        t[0] += w[u].v[i] * e[u].v[i];
        if (LAYER) t[1] += w[u].v[i];
      }
    }
    s[0] += c.skip[u] < kGroup ? t[0] : 0.0f;
    if (LAYER) s[1] += c.skip[u] < kGroup ? t[1] : 0.0f;
  }
}

// Mean and 1 / sqrt(variance + eps) of a team's row.
template <int U, bool LAYER, bool SMALL>
__device__ __forceinline__ void row_stats(const Vec8 (&v)[U], const Columns<U>& c, int lanes,
                                          float inv_cols, float eps, float* slots, float* mean,
                                          float* rstd) {
  float s[1] = {0.0f};
  *mean = 0.0f;
  if (LAYER) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) s[0] += i >= c.skip[u] ? v[u].v[i] : 0.0f;
    }
    team_sum<1, SMALL>(s, lanes, slots);
    *mean = s[0] * inv_cols;
    s[0] = 0.0f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const float d = v[u].v[i] - *mean;
      s[0] += i >= c.skip[u] ? d * d : 0.0f;
    }
  }
  team_sum<1, SMALL>(s, lanes, slots + 16);
  *rstd = 1.0f / sqrtf(s[0] * inv_cols + eps);
}

struct Forward {
  const void *x, *residual, *post, *post_bias, *pre, *pre_bias, *gate;
  void *h, *y;
  float* stats;
  int64_t rows;
  int cols;
  int64_t rows_per_gate;
  float scale, offset, eps, inv_cols;
  int lanes, teams;
};

template <typename T, int U, bool LAYER, int THREADS>
__global__ __launch_bounds__(THREADS) void block_norms(Forward a) {
  constexpr bool kSmall = U == 1;
  // Two sets of slots, for the rounds in turn: a barrier lies between a read
  // and the next write of the same set.
  __shared__ float slots[2][64];
  const int team = threadIdx.x / a.lanes;
  const Columns<U> c = columns_of<U>(threadIdx.x % a.lanes, a.lanes, a.cols);
  int set = 0;
  const T* post = static_cast<const T*>(a.post);
  const T* pre = static_cast<const T*>(a.pre);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * a.teams; first < a.rows;
       first += static_cast<int64_t>(gridDim.x) * a.teams, set ^= 1) {
    const bool valid = first + team < a.rows;
    const int64_t row = valid ? first + team : a.rows - 1;
    const int64_t at = row * a.cols;
    Vec8 n[U], h[U];
#pragma unroll
    for (int u = 0; u < U; ++u) n[u] = load8_once(static_cast<const T*>(a.x) + at + c.col[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      h[u] = load8_once(static_cast<const T*>(a.residual) + at + c.col[u]);
    }
    float mean0 = 0.0f, rstd0 = 1.0f, mean1 = 0.0f, rstd1 = 1.0f;
    if (post) {
      row_stats<U, LAYER, kSmall>(n, c, a.lanes, a.inv_cols, a.eps, slots[set], &mean0, &rstd0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Vec8 w = load8(post + c.col[u]);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          n[u].v[i] = (n[u].v[i] - mean0) * rstd0 * (a.offset + w.v[i]);
        }
        if (a.post_bias) {
          const Vec8 b = load8(static_cast<const T*>(a.post_bias) + c.col[u]);
#pragma unroll
          for (int i = 0; i < kGroup; ++i) n[u].v[i] += b.v[i];
        }
      }
    }
    const T* gate =
        a.gate ? static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.cols : nullptr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (gate) {
        const Vec8 g = load8(gate + c.col[u]);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) n[u].v[i] *= g.v[i];
      }
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        h[u].v[i] = as_stored(__builtin_fmaf(a.scale, n[u].v[i], h[u].v[i]), post);
      }
      if (valid && c.skip[u] < kGroup) store8<true>(static_cast<T*>(a.h) + at + c.col[u], h[u]);
    }
    if (pre) {
      row_stats<U, LAYER, kSmall>(h, c, a.lanes, a.inv_cols, a.eps, slots[set] + 32, &mean1,
                                  &rstd1);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Vec8 w = load8(pre + c.col[u]);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          h[u].v[i] = (h[u].v[i] - mean1) * rstd1 * (a.offset + w.v[i]);
        }
        if (a.pre_bias) {
          const Vec8 b = load8(static_cast<const T*>(a.pre_bias) + c.col[u]);
#pragma unroll
          for (int i = 0; i < kGroup; ++i) h[u].v[i] += b.v[i];
        }
        if (valid && c.skip[u] < kGroup) store8<true>(static_cast<T*>(a.y) + at + c.col[u], h[u]);
      }
    }
    if (valid && threadIdx.x % a.lanes == 0) {
      *reinterpret_cast<f32x4_a4_t*>(a.stats + row * 4) = f32x4_t{mean0, rstd0, mean1, rstd1};
    }
  }
}

// Column sums of the gradient, in the order of the join's outputs.
enum Sum { kPre, kPreBias, kPost, kPostBias, kGate, kSums };

struct Backward {
  const void *grad_h, *grad_y, *x, *h;
  const float* stats;
  const void *post, *post_bias, *pre, *gate;
  void *dx, *dresidual, *dgate;
  float* part;  // [kSums][blocks][cols], kGate: [2 blocks][cols] at the end
  int64_t rows;
  int cols;
  int64_t rows_per_gate;
  float scale, offset, inv_cols;
  int lanes, teams, blocks;
};

__device__ __forceinline__ int64_t first_row(int64_t rows, int block, int blocks) {
  return rows * block / blocks;
}

// A workgroup takes consecutive rows, its teams in turn, and keeps the column
// sums of all of them in registers; the rows of one gate are a segment, whose
// sum goes out when the segment ends: as dgate where the segment holds all rows
// of the gate, else to one of the workgroup's two places for the join (a
// workgroup has at most two such segments, its first and its last).
// With one group a lane the next row's operands are loaded before the current
// one's are used.
enum Gate { kNoGate, kGateOfRows, kGateByRow };  // none, shared by rows, one a row

template <typename T, int U, bool SMALL, bool LAYER, bool PRE, bool POST, Gate GATE, int THREADS>
__global__ __launch_bounds__(THREADS) void block_norms_bwd(Backward a) {
  constexpr bool kSmall = SMALL;
  constexpr bool kAhead = U == 1;  // with two groups a lane has no registers for it
  // 16 waves leave a lane 128 registers.  The two weights' sums then lie in LDS, 128
  // KB of it, read and written once a row (16 bytes of a lane beside the next's), and
  // weights and gate are loaded where they are used: [4096, 12288] bf16 297 -> 151 us.
  // Of 512 threads not: [8192, 5120] 115 -> 125 us (122 with the next row's loads ahead,
  // for which there is room then), [8192, 8192] 148 -> 153 (159), with a gate a row
  // 216 -> 218 (241).  Biases' and gates' sums still spill: of LayerNorm before and
  // after the sum 52 registers a lane, with a gate a row 88, with one that rows share
  // 194 ([4096, 16384] with 16 gates 607 us, where RMSNorm without a gate, which spills
  // none, takes 177); of 512 threads the last alone, 29 ([8192, 8192] 245 and 148).
  constexpr bool kFewRegisters = THREADS == 1024;
  __shared__ float slots[2][64];
  __shared__ f32x4_t held[kFewRegisters ? 2 * U * 2 * THREADS : 1];
  extern __shared__ float sums[];  // [teams][cols], where there are several teams
  const int team = threadIdx.x / a.lanes;
  const Columns<U> c = columns_of<U>(threadIdx.x % a.lanes, a.lanes, a.cols);
  const int64_t begin = first_row(a.rows, blockIdx.x, a.blocks);
  const int64_t end = first_row(a.rows, blockIdx.x + 1, a.blocks);
  Vec8 acc[kSums][U];
  auto sum_of = [&](int k, int u) __attribute__((always_inline)) {
    if (!kFewRegisters || (k != kPre && k != kPost)) return acc[k][u];
    const f32x4_t* at = held + ((k == kPost) * U + u) * 2 * THREADS + threadIdx.x;
    const f32x4_t v = at[0], w = at[THREADS];
    return Vec8{{v[0], v[1], v[2], v[3], w[0], w[1], w[2], w[3]}};
  };
  auto set_sum = [&](int k, int u, const Vec8& v) __attribute__((always_inline)) {
    if (!kFewRegisters || (k != kPre && k != kPost)) {
      acc[k][u] = v;
      return;
    }
    f32x4_t* at = held + ((k == kPost) * U + u) * 2 * THREADS + threadIdx.x;
    at[0] = f32x4_t{v.v[0], v.v[1], v.v[2], v.v[3]};
    at[THREADS] = f32x4_t{v.v[4], v.v[5], v.v[6], v.v[7]};
  };
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
#pragma unroll
    for (int u = 0; u < U; ++u) set_sum(k, u, Vec8{});
  }
  // (In registers where there is room, as a load in the loop would wait for the next
  // row's.)
  Vec8 wpre[U], wpost[U], bpost[U], gate[U];
  auto vector = [&](Vec8 (&w)[U], const void* from, float plus) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = load8(static_cast<const T*>(from) + c.col[u]);
#pragma unroll
      for (int i = 0; i < kGroup; ++i) w[u].v[i] += plus;
    }
  };
  auto load_pre = [&]() __attribute__((always_inline)) { vector(wpre, a.pre, a.offset); };
  auto load_post = [&]() __attribute__((always_inline)) {
    vector(wpost, a.post, a.offset);
    if (GATE && LAYER) {
      if (a.post_bias) {
        vector(bpost, a.post_bias, 0.0f);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) bpost[u] = Vec8{};
      }
    }
  };
  // scale * gate of one of its rows.
  auto load_gate = [&](int64_t which) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      gate[u] = load8(static_cast<const T*>(a.gate) + which * a.cols + c.col[u]);
#pragma unroll
      for (int i = 0; i < kGroup; ++i) gate[u].v[i] *= a.scale;
    }
  };
  if (!kFewRegisters && PRE) load_pre();
  if (!kFewRegisters && POST) load_post();

  // The sum over the teams of one accumulator, written by put(column, value).
  auto flush = [&](Vec8 (&v)[U], auto put) {
    if (a.teams > 1) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          if (i >= c.skip[u]) sums[team * a.cols + c.col[u] + i] = v[u].v[i];
        }
      }
      __syncthreads();
      for (int j = threadIdx.x; j < a.cols; j += blockDim.x) {
        float s = 0.0f;
        for (int t = 0; t < a.teams; ++t) s += sums[t * a.cols + j];
        put(j, s);
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          if (i >= c.skip[u]) put(c.col[u] + i, v[u].v[i]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = Vec8{};
  };

  int set = 0;
  const bool ragged = a.cols % kGroup != 0;
  constexpr bool by_row = GATE == kGateByRow;
  for (int64_t from = begin; from < end;) {
    int64_t to = end, which = 0;
    if (GATE && !by_row) {
      which = from / a.rows_per_gate;
      to = min(end, (which + 1) * a.rows_per_gate);
      if (!kFewRegisters) load_gate(which);
    }
    // All loads without a branch, or the compiler waits for them at its end.
    const T* grad_h = static_cast<const T*>(a.grad_h ? a.grad_h : a.grad_y);
    struct Row {
      Raw8<T> gh[U], gy[U], h[U], x[U], gate[U];
      float st[4];
    };
    auto load = [&](Row& next, int64_t first) __attribute__((always_inline)) {
      const int64_t row = min(first + team, to - 1);
      const int64_t at = row * a.cols;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (PRE) next.gy[u].load_once(static_cast<const T*>(a.grad_y) + at + c.col[u]);
        if (PRE) next.h[u].load_once(static_cast<const T*>(a.h) + at + c.col[u]);
        next.gh[u].load_once(grad_h + at + c.col[u]);
        if (POST || GATE) next.x[u].load_once(static_cast<const T*>(a.x) + at + c.col[u]);
        if (by_row && !kFewRegisters) {
          next.gate[u].load_once(static_cast<const T*>(a.gate) + at + c.col[u]);
        }
      }
      // (What is not used is not loaded: its register would be waited for.)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((i < 2 ? POST : PRE) && (LAYER || i % 2 == 1)) next.st[i] = a.stats[row * 4 + i];
      }
    };
    auto step = [&](Row& row, Row& next, int64_t first) __attribute__((always_inline)) {
      const bool valid = first + team < to;
      const int64_t at = (first + team) * a.cols;
      if (!kAhead) load(row, first);
      Vec8 gh[U], gy[U], h[U], x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // A team past the last row adds nothing: its gradients are 0.
        row.gy[u].clear_unless(valid);
        row.gh[u].clear_unless(valid && a.grad_h);
        if (PRE) gy[u] = row.gy[u].values();
        if (PRE) h[u] = row.h[u].values();
        gh[u] = row.gh[u].values();
        if (by_row && !kFewRegisters) {
          gate[u] = row.gate[u].values();
#pragma unroll
          for (int i = 0; i < kGroup; ++i) gate[u].v[i] *= a.scale;
        }
      }
      const float st[4] = {row.st[0], row.st[1], row.st[2], row.st[3]};
      if (kAhead) load(next, min(first + a.teams, to - 1));
      // gh becomes T.
      if (PRE) {
        if (kFewRegisters) load_pre();
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Vec8 dw = sum_of(kPre, u), db = sum_of(kPreBias, u);
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            h[u].v[i] = (LAYER ? h[u].v[i] - st[2] : h[u].v[i]) * st[3];
            dw.v[i] += gy[u].v[i] * h[u].v[i];
            db.v[i] += gy[u].v[i];
            gy[u].v[i] *= wpre[u].v[i];
          }
          set_sum(kPre, u, dw);
          if (LAYER) set_sum(kPreBias, u, db);
        }
        float s[2] = {0.0f, 0.0f};
        pair_sum<U, LAYER>(s, gy, h, c, ragged);
        team_sum<LAYER ? 2 : 1, kSmall>(s, a.lanes, slots[set]);
        s[0] *= st[3] * a.inv_cols;
        s[1] *= st[3] * a.inv_cols;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            const float rest = LAYER ? gh[u].v[i] - s[1] : gh[u].v[i];
            gh[u].v[i] = __builtin_fmaf(st[3], gy[u].v[i], __builtin_fmaf(-h[u].v[i], s[0], rest));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (valid && c.skip[u] < kGroup) {
          store8(static_cast<T*>(a.dresidual) + at + c.col[u], gh[u]);
        }
      }
      // gh becomes v = scale gate T, x the normalised x.
      if (kFewRegisters && POST) load_post();
      if (kFewRegisters && GATE) load_gate(by_row ? min(first + team, to - 1) : which);
      if (POST || GATE) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Vec8 tn;
          x[u] = row.x[u].values();
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            float n = x[u].v[i];
            if (POST) {
              x[u].v[i] = (LAYER ? n - st[0] : n) * st[1];
              n = x[u].v[i] * wpost[u].v[i];
              if (LAYER) n = __builtin_fmaf(x[u].v[i], wpost[u].v[i], bpost[u].v[i]);
            }
            if (GATE == kGateOfRows) acc[kGate][u].v[i] += gh[u].v[i] * n;
            tn.v[i] = gh[u].v[i] * n * a.scale;
          }
          if (by_row && valid && c.skip[u] < kGroup) {
            store8(static_cast<T*>(a.dgate) + at + c.col[u], tn);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        Vec8 dw = sum_of(kPost, u), db = sum_of(kPostBias, u);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          gh[u].v[i] *= GATE ? gate[u].v[i] : a.scale;
          if (POST) {
            dw.v[i] += gh[u].v[i] * x[u].v[i];
            db.v[i] += gh[u].v[i];
            gh[u].v[i] *= wpost[u].v[i];
          }
        }
        if (POST) set_sum(kPost, u, dw);
        if (POST && LAYER) set_sum(kPostBias, u, db);
      }
      if (POST) {
        float s[2] = {0.0f, 0.0f};
        pair_sum<U, LAYER>(s, gh, x, c, ragged);
        team_sum<LAYER ? 2 : 1, kSmall>(s, a.lanes, slots[set] + 32);
        s[0] *= st[1] * a.inv_cols;
        s[1] *= st[1] * a.inv_cols;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            const float rest = x[u].v[i] * -s[0];
            gh[u].v[i] =
                __builtin_fmaf(st[1], gh[u].v[i], LAYER ? rest - s[1] : rest);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (valid && c.skip[u] < kGroup) store8(static_cast<T*>(a.dx) + at + c.col[u], gh[u]);
      }
      set ^= 1;
    };
    // Two sets of registers in turn: one would be copied, which waits for it.
    Row even, odd;
    if (kAhead) load(even, from);
    for (int64_t first = from; first < to; first += a.teams) {
      step(even, odd, first);
      first += a.teams;
      if (first >= to) break;
      step(odd, even, first);
    }
    if (GATE && !by_row) {
      const bool whole = from == which * a.rows_per_gate && to == (which + 1) * a.rows_per_gate;
      if (whole) {
        T* out = static_cast<T*>(a.dgate) + which * a.cols;
        flush(acc[kGate], [&](int j, float s) { store1(out + j, s * a.scale); });
      } else {
        float* out = a.part + (static_cast<int64_t>(kGate) * a.blocks + 2 * blockIdx.x +
                               (from == begin ? 0 : 1)) * a.cols;
        flush(acc[kGate], [&](int j, float s) { out[j] = s * a.scale; });
      }
    }
    from = to;
  }
  auto put_part = [&](int k) __attribute__((always_inline)) {
    Vec8 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = sum_of(k, u);
    float* out = a.part + (static_cast<int64_t>(k) * a.blocks + blockIdx.x) * a.cols;
    flush(v, [&](int j, float s) { out[j] = s; });
  };
  if (PRE) put_part(kPre);
  if (PRE && LAYER) put_part(kPreBias);
  if (POST) put_part(kPost);
  if (POST && LAYER) put_part(kPostBias);
}

struct Join {
  const float* part;
  void* out[kSums];
  int64_t rows;
  int cols;
  int64_t rows_per_gate;
  int blocks;
  bool by_boundary;
};

// The workgroup that row `row` falls to.
__device__ __forceinline__ int block_of(int64_t row, int64_t rows, int blocks) {
  int b = static_cast<int>(row * blocks / rows);
  while (b + 1 < blocks && first_row(rows, b + 1, blocks) <= row) ++b;
  return b;
}

// The workgroups' column sums added in their order: 32 columns by 32 parts of
// the workgroups, the parts joined through LDS.  blockIdx.y: one of the four
// sums over all rows, or from 4 on a gate: each, or (`by_boundary`, where there
// are more gates than workgroups) the one that the boundary behind a workgroup
// lies in, where it is the first in that gate.
template <typename T>
__global__ __launch_bounds__(1024) void join_sums(Join a) {
  __shared__ float parts[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x % 32;
  const int part = threadIdx.x / 32;
  const int k = min(static_cast<int>(blockIdx.y), static_cast<int>(kGate));
  if (!a.out[k]) return;
  int lo = 0, hi = a.blocks;
  int64_t gate = 0;
  bool second = false;  // whether workgroup `lo` has the gate as its last segment
  if (k == kGate) {
    const int at = blockIdx.y - kGate;
    gate = a.by_boundary ? first_row(a.rows, at + 1, a.blocks) / a.rows_per_gate : at;
    const int64_t from = gate * a.rows_per_gate;
    lo = block_of(from, a.rows, a.blocks);
    hi = block_of(from + a.rows_per_gate - 1, a.rows, a.blocks) + 1;
    // Within one workgroup: written there.  Another boundary is the gate's first.
    if (hi == lo + 1 || (a.by_boundary && lo != at)) return;
    second = first_row(a.rows, lo, a.blocks) < from;
  }
  float s = 0.0f;
  if (col < a.cols) {
    // kGate: two places a workgroup, the first for the segment it begins with.
    const int64_t step = k == kGate ? 2 * a.cols : a.cols;
    const float* p = a.part + static_cast<int64_t>(k) * a.blocks * a.cols + col;
    const int n = hi - lo, end = n * (part + 1) / 32;
#pragma unroll 4
    for (int b = n * part / 32; b < end; ++b) {
      s += p[(lo + b) * step + (b == 0 && second ? a.cols : 0)];
    }
  }
  parts[part][threadIdx.x % 32] = s;
  __syncthreads();
  if (part == 0 && col < a.cols) {
    s = 0.0f;
    for (int i = 0; i < 32; ++i) s += parts[i][threadIdx.x];
    store1(static_cast<T*>(a.out[k]) + gate * a.cols + col, s);
  }
}

int check_sizes(const char* what, int elem_size, int64_t rows, int64_t cols, int64_t gates,
                int layer, const void* post, const void* post_bias, const void* pre,
                const void* pre_bias, const void* gate, float scale, float offset) {
  HIPO_REQUIRE(elem_size == 2 || elem_size == 4, "%s: elem_size must be 2 or 4", what);
  HIPO_REQUIRE(rows >= 0 && cols >= 0 && gates >= 0, "%s: negative size", what);
  HIPO_REQUIRE(cols >= kGroup && cols <= kMostCols, "%s: cols must be from 8 to 16384", what);
  HIPO_REQUIRE(rows < (int64_t{1} << 31), "%s: rows must be below 2^31", what);
  HIPO_REQUIRE(layer == 0 || layer == 1, "%s: layer must be 0 or 1", what);
  HIPO_REQUIRE(post || pre, "%s: a norm is needed before or after the sum", what);
  HIPO_REQUIRE((post || !post_bias) && (pre || !pre_bias), "%s: a bias needs its norm", what);
  HIPO_REQUIRE(layer || (!post_bias && !pre_bias), "%s: biases are LayerNorm's", what);
  HIPO_REQUIRE((gates > 0) == (gate != nullptr), "%s: gate and gate_rows go together", what);
  HIPO_REQUIRE(gates == 0 || rows % gates == 0, "%s: gate_rows must divide rows", what);
  HIPO_REQUIRE(__builtin_isfinite(scale) && __builtin_isfinite(offset),
               "%s: scale and offset must be finite", what);
  return 0;
}

template <typename T, int U, int THREADS>
void launch_fwd(const Forward& a, bool layer, int64_t blocks, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(blocks)), block(a.lanes * a.teams);
  if (layer) {
    block_norms<T, U, true, THREADS><<<grid, block, 0, stream>>>(a);
  } else {
    block_norms<T, U, false, THREADS><<<grid, block, 0, stream>>>(a);
  }
}

template <typename T>
int run_fwd(const Forward& a, bool layer, hipStream_t stream) {
  const int64_t blocks = std::min<int64_t>((a.rows + a.teams - 1) / a.teams, int64_t{1} << 20);
  if (a.cols <= kSmallCols) {
    launch_fwd<T, 1, 512>(a, layer, blocks, stream);
  } else if (a.lanes * a.teams <= 512) {
    launch_fwd<T, 2, 512>(a, layer, blocks, stream);
  } else {
    launch_fwd<T, 2, 1024>(a, layer, blocks, stream);
  }
  return check_launch("block_norms");
}

template <typename T, int U, bool SMALL, bool LAYER, bool PRE, bool POST, int THREADS>
void launch_bwd(const Backward& a, hipStream_t stream) {
  const dim3 grid(a.blocks), block(a.lanes * a.teams);
  const size_t lds = a.teams > 1 ? sizeof(float) * a.teams * a.cols : 0;
  if (!a.gate) {
    block_norms_bwd<T, U, SMALL, LAYER, PRE, POST, kNoGate, THREADS>
        <<<grid, block, lds, stream>>>(a);
  } else if (a.rows_per_gate == 1) {
    block_norms_bwd<T, U, SMALL, LAYER, PRE, POST, kGateByRow, THREADS>
        <<<grid, block, lds, stream>>>(a);
  } else {
    block_norms_bwd<T, U, SMALL, LAYER, PRE, POST, kGateOfRows, THREADS>
        <<<grid, block, lds, stream>>>(a);
  }
}

template <typename T, int U, bool SMALL, int THREADS>
void launch_bwd(const Backward& a, bool layer, hipStream_t stream) {
  if (a.pre && a.post) {
    layer ? launch_bwd<T, U, SMALL, true, true, true, THREADS>(a, stream)
          : launch_bwd<T, U, SMALL, false, true, true, THREADS>(a, stream);
  } else if (a.pre) {
    layer ? launch_bwd<T, U, SMALL, true, true, false, THREADS>(a, stream)
          : launch_bwd<T, U, SMALL, false, true, false, THREADS>(a, stream);
  } else {
    layer ? launch_bwd<T, U, SMALL, true, false, true, THREADS>(a, stream)
          : launch_bwd<T, U, SMALL, false, false, true, THREADS>(a, stream);
  }
}

// Workgroups of the gradient: no more than there are rows for their teams, and one a
// CU.  Two were, RMSNorm before and after the sum of 8192 rows: of 1280 columns 32.1 ->
// 31.1 us, 2560 55.7 -> 53.2, 2880 61.1 -> 60.7, but 3584 69.2 -> 72.3, 4096 74.3 ->
// 78.5, 5120 115 -> 123, 8192 148 -> 167, and 16384 x 2880 with 16 gates 126 -> 138:
// twice the sums to write and join, and few variants fit a CU twice.
int bwd_blocks(int64_t rows, int64_t cols) {
  const Layout l = layout_of(cols, bwd_groups(cols));
  return static_cast<int>(std::min<int64_t>((rows + l.teams - 1) / l.teams, 256));
}

template <typename T>
int run_bwd(const Backward& a, Join j, bool layer, hipStream_t stream) {
  if (a.cols <= kSmallCols) {
    launch_bwd<T, 1, true, 512>(a, layer, stream);
  } else if (bwd_groups(a.cols) == 1) {
    launch_bwd<T, 1, false, 512>(a, layer, stream);
  } else if (a.lanes * a.teams <= 512) {
    launch_bwd<T, 2, false, 512>(a, layer, stream);
  } else {
    launch_bwd<T, 2, false, 1024>(a, layer, stream);
  }
  const int rc = check_launch("block_norms_bwd");
  if (rc != 0) return rc;
  // Gates whose rows may lie in several workgroups.
  int64_t gates = a.gate && a.rows_per_gate != 1 ? a.rows / a.rows_per_gate : 0;
  j.by_boundary = gates > a.blocks;
  gates = std::min<int64_t>(gates, j.by_boundary ? a.blocks - 1 : gates);
  join_sums<T><<<dim3((a.cols + 31) / 32, static_cast<uint32_t>(kGate + gates)), 1024, 0,
                 stream>>>(j);
  return check_launch("block_norms_bwd: join_sums");
}

}  // namespace
}  // namespace hipo

extern "C" int hipo_block_norms(const void* x, const void* residual, int elem_size,
                                const void* post, const void* post_bias, const void* pre,
                                const void* pre_bias, const void* gate, void* h, void* y,
                                float* stats, int64_t rows, int64_t cols, int64_t gate_rows,
                                float scale, float offset, float eps, int layer,
                                hipStream_t stream) {
  using namespace hipo;
  clear_error();
  const int rc = check_sizes("block_norms", elem_size, rows, cols, gate_rows, layer, post,
                             post_bias, pre, pre_bias, gate, scale, offset);
  if (rc != 0) return rc;
  HIPO_REQUIRE(eps >= 0.0f && __builtin_isfinite(eps),
               "block_norms: eps must be finite, not negative");
  if (rows == 0) return 0;
  HIPO_REQUIRE(x && residual && h && stats && (y || !pre), "block_norms: null pointer");
  const Layout l = layout_of(cols, 2);
  const Forward a{x, residual, post, post_bias, pre, pre_bias, gate, h, y, stats, rows,
                  static_cast<int>(cols), gate_rows ? rows / gate_rows : rows, scale, offset, eps,
                  1.0f / static_cast<float>(cols), l.lanes, l.teams};
  return elem_size == 2 ? run_fwd<uint16_t>(a, layer != 0, stream)
                        : run_fwd<float>(a, layer != 0, stream);
}

extern "C" size_t hipo_block_norms_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols < hipo::kGroup || cols > hipo::kMostCols) return 0;
  return sizeof(float) * (hipo::kSums + 1) * hipo::bwd_blocks(rows, cols) * cols;
}

extern "C" int hipo_block_norms_bwd(const void* grad_h, const void* grad_y, const void* x,
                                    const void* h, const float* stats, int elem_size,
                                    const void* post, const void* post_bias, const void* pre,
                                    const void* pre_bias, const void* gate, void* dx,
                                    void* dresidual, void* dgate, void* dpost, void* dpost_bias,
                                    void* dpre, void* dpre_bias, int64_t rows, int64_t cols,
                                    int64_t gate_rows, float scale, float offset, int layer,
                                    void* workspace, size_t workspace_bytes,
                                    hipStream_t stream) {
  using namespace hipo;
  clear_error();
  const char* what = "block_norms_bwd";
  const int rc = check_sizes(what, elem_size, rows, cols, gate_rows, layer, post, post_bias, pre,
                             pre_bias, gate, scale, offset);
  if (rc != 0) return rc;
  HIPO_REQUIRE((pre || !grad_y) && (pre || grad_h), "%s: grad_y belongs to the norm after the sum",
               what);
  HIPO_REQUIRE((dpost != nullptr) == (post != nullptr) && (dpre != nullptr) == (pre != nullptr) &&
                   (dpost_bias != nullptr) == (post_bias != nullptr) &&
                   (dpre_bias != nullptr) == (pre_bias != nullptr),
               "%s: each weight and bias has its gradient", what);
  if (rows == 0) return 0;
  HIPO_REQUIRE(stats && dx && dresidual && (x || !(post || gate)) && ((h && grad_y) || !pre) &&
                   (dgate != nullptr) == (gate != nullptr),
               "%s: null pointer", what);
  const size_t need = hipo_block_norms_bwd_workspace_bytes(rows, cols);
  HIPO_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
               "%s: workspace of %zu bytes, 16-byte aligned, needed", what, need);
  const Layout l = layout_of(cols, bwd_groups(cols));
  const int64_t rows_per_gate = gate_rows ? rows / gate_rows : rows;
  const int blocks = bwd_blocks(rows, cols);
  const Backward a{grad_h, grad_y, x, h, stats, post, post_bias, pre, gate, dx, dresidual, dgate,
                   static_cast<float*>(workspace), rows, static_cast<int>(cols), rows_per_gate,
                   scale, offset, 1.0f / static_cast<float>(cols), l.lanes, l.teams, blocks};
  const Join j{a.part, {dpre, dpre_bias, dpost, dpost_bias, rows_per_gate == 1 ? nullptr : dgate},
               rows, a.cols, rows_per_gate, blocks, false};
  return elem_size == 2 ? run_bwd<uint16_t>(a, j, layer != 0, stream)
                        : run_bwd<float>(a, j, layer != 0, stream);
}
