// Embedding lookup with a scale, and its gradient:
//   out[t] = scale * w[token_t],    dw[v] = scale * sum_{t: token_t = v} grad[t],
// the sum in fp32 in an order that the tokens alone fix, one rounding at the
// end.  Both move rows: HBM bounds them.
//
// Lookup: a lane per 16-byte piece of the output, pieces in memory order, so
// no lane is idle whatever the width.
//
// Gradient, three launches:
//   1. sort_tokens: the positions in order of their token, equal tokens in
//      order of position.  A workgroup owns the tokens with one remainder
//      modulo the number of workgroups (a vocabulary is ordered by frequency:
//      ranges of it would give one workgroup most of the tokens) and scans all
//      tokens twice, for the counts and for the places: no exchange between
//      workgroups, no atomics on memory, and the scan is a small part of
//      reading the gradient rows (8 bytes of a token from the L2 against
//      hundreds to thousands).
//   2. sum_pieces: tokens that occur more than kPiece times are cut into
//      pieces of kPiece positions, each summed on its own (fp32, into the
//      workspace).
//   3. write_rows: a lane per piece of columns of a row of dw: the sum of its
//      few positions, or of its pieces, or zeros.  Adding into dw only visits
//      rows that have a token.
#include <math.h>

#include <algorithm>

#include "hipo_common.h"

namespace hipo {
namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortLoads = 8;        // tokens per thread in flight
constexpr int kSortRows = 512;       // rows of dw per sorting workgroup
constexpr int kSortRowBits = 9;
constexpr int kSortGroups = 256;     // at least: one workgroup per CU
constexpr int kPiece = 64;           // positions per piece of a frequent token
constexpr int64_t kLanes = int64_t{1} << 30;  // lanes per launch

typedef uint16_t u16x4_t __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ int64_t token_at(const void* tokens, int size, int64_t i) {
  return size == 8 ? static_cast<const int64_t*>(tokens)[i]
                   : static_cast<const int32_t*>(tokens)[i];
}

// C consecutive values at any element alignment, as they lie in memory.
template <typename T, int C>
struct Values {
  typedef T Vec __attribute__((ext_vector_type(C)));
  typedef Vec Unaligned __attribute__((aligned(sizeof(T))));
  static_assert(sizeof(Vec) <= 16 && (sizeof(Vec) & (sizeof(Vec) - 1)) == 0, "one access");
  Vec v;

  __device__ __forceinline__ void load(const T* p) {
    v = *reinterpret_cast<const Unaligned*>(p);
  }
  __device__ __forceinline__ void load_stream(const T* p) {
    v = __builtin_nontemporal_load(reinterpret_cast<const Unaligned*>(p));
  }
  __device__ __forceinline__ void store_stream(T* p) const {
    __builtin_nontemporal_store(v, reinterpret_cast<Unaligned*>(p));
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Unaligned*>(p) = v; }
  // The first n of them, one by one.
  __device__ __forceinline__ void load_part(const T* p, int n) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = i < n ? p[i] : T{0};
  }
  __device__ __forceinline__ void store_part(T* p, int n) const {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (i < n) p[i] = v[i];
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 2) return bf16_to_f32(v[i]);
    else return v[i];
  }
  __device__ __forceinline__ void set(const float (&f)[C]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < C; i += 2) {
        const uint32_t w = pack_bf16x2(f[i], f[i + 1]);
        v[i] = static_cast<T>(w & 0xffffu);
        v[i + 1] = static_cast<T>(w >> 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = f[i];
    }
  }
};

struct FwdArgs {
  const void* w;
  const void* tokens;
  void* out;
  int64_t first, count, vocab, row_stride;  // tokens [first, first + count)
  DivMagic by_pieces;
  int width, pieces;  // pieces of C values per row
  float scale;
  int token_size;
};

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void embedding_rows(FwdArgs a) {
  constexpr int C = 16 / sizeof(T);
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = div_by(id, a.by_pieces);
  if (t >= a.count) return;
  const int col = static_cast<int>(id - t * a.pieces) * C;
  const int64_t v = token_at(a.tokens, a.token_size, a.first + t);
  const bool known = v >= 0 && v < a.vocab;
  const T* w = static_cast<const T*>(a.w) + (known ? v : 0) * a.row_stride + col;
  T* out = static_cast<T*>(a.out) + (a.first + t) * a.width + col;
  const int left = a.width - col;
  Values<T, C> x;
  if (WHOLE || left >= C) x.load(w);
  else x.load_part(w, left);
  float f[C];
#pragma unroll
  for (int i = 0; i < C; ++i) f[i] = known ? x.get(i) * a.scale : __builtin_nanf("");
  x.set(f);
  if (WHOLE || left >= C) x.store_stream(out);
  else x.store_part(out, left);
}

// Where a row's positions are in the sorted order.
struct Segment {
  int start, count;
};
struct Place {
  int position, row;
};

struct SortArgs {
  const void* tokens;
  Segment* segments;  // [vocab]
  Place* order;       // [count]
  int* total;         // tokens that count
  int64_t count, vocab, padding_idx;
  int token_size, group_bits;  // 2^group_bits workgroups
};

__global__ __launch_bounds__(kSortThreads) void sort_tokens(SortArgs a) {
  __shared__ int next[kSortRows];                          // count, then next place
  __shared__ unsigned short seen[kSortWaves][kSortRows];   // a batch's counts per wave
  __shared__ int wave_sum_[kSortWaves];
  __shared__ int wave_below[kSortWaves];
  __shared__ int found[kSortLoads * kSortWaves];
  __shared__ int list_row[kSortLoads * kSortThreads];
  __shared__ int list_pos[kSortLoads * kSortThreads];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int groups = 1 << a.group_bits;
  const int mine = blockIdx.x;
  for (int i = tid; i < kSortRows; i += kSortThreads) next[i] = 0;
  for (int i = tid; i < kSortWaves * kSortRows; i += kSortThreads) (&seen[0][0])[i] = 0;
  __syncthreads();

  // -1: does not count.
  const auto row_of = [&](int64_t i) -> int64_t {
    if (i >= a.count) return -1;
    const int64_t v = token_at(a.tokens, a.token_size, i);
    return v >= 0 && v < a.vocab && v != a.padding_idx ? v : -1;
  };

  int below = 0;
  for (int64_t i0 = 0; i0 < a.count; i0 += kSortLoads * kSortThreads) {
    int64_t v[kSortLoads];
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) v[u] = row_of(i0 + u * kSortThreads + tid);
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) {
      if (v[u] < 0) continue;
      const int g = static_cast<int>(v[u] & (groups - 1));
      below += g < mine;
      if (g == mine) atomicAdd(&next[v[u] >> a.group_bits], 1);
    }
  }
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) below += __shfl_xor(below, d);
  if (lane == 0) wave_below[wave] = below;
  __syncthreads();

  // Exclusive sums of the counts, one row per thread.
  const int n = tid < kSortRows ? next[tid] : 0;
  int sum = n;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == kWave - 1) wave_sum_[wave] = sum;
  __syncthreads();
  int start = sum - n;
  for (int w = 0; w < kSortWaves; ++w) {
    start += wave_below[w];
    if (w < wave) start += wave_sum_[w];
  }
  if (tid < kSortRows) {
    next[tid] = start;
    const int64_t row = (static_cast<int64_t>(tid) << a.group_bits) + mine;
    if (row < a.vocab) a.segments[row] = Segment{start, n};
    if (mine == groups - 1 && tid == kSortRows - 1) *a.total = start + n;
  }
  __syncthreads();

  for (int64_t i0 = 0; i0 < a.count; i0 += kSortLoads * kSortThreads) {
    // This batch's tokens, in order of position, into the list.
    int row[kSortLoads], before[kSortLoads];
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) {
      const int64_t v = row_of(i0 + u * kSortThreads + tid);
      row[u] = v >= 0 && (v & (groups - 1)) == mine ? static_cast<int>(v >> a.group_bits) : -1;
    }
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) {
      const uint64_t m = __ballot(row[u] >= 0);
      before[u] = __popcll(m & ((uint64_t{1} << lane) - 1));
      if (lane == 0) found[u * kSortWaves + wave] = __popcll(m);
    }
    __syncthreads();
    int total = 0;
    {
      int at[kSortLoads];
#pragma unroll
      for (int u = 0; u < kSortLoads; ++u) {
        for (int w = 0; w < kSortWaves; ++w) {
          if (w == wave) at[u] = total;
          total += found[u * kSortWaves + w];
        }
      }
#pragma unroll
      for (int u = 0; u < kSortLoads; ++u) {
        if (row[u] < 0) continue;
        list_row[at[u] + before[u]] = row[u];
        list_pos[at[u] + before[u]] = static_cast<int>(i0) + u * kSortThreads + tid;
      }
    }
    __syncthreads();
    // Places: after what came before in the tokens, the waves before in this
    // round of 1024, and the lanes before with the same row.
    for (int l0 = 0; l0 < total; l0 += kSortThreads) {
      const int i = l0 + tid;
      const bool in = i < total;
      const int r = in ? list_row[i] : -1;
      uint64_t same = __ballot(in);
#pragma unroll
      for (int b = 0; b < kSortRowBits; ++b) {
        const uint64_t m = __ballot((r >> b) & 1);
        same &= ((r >> b) & 1) ? m : ~m;
      }
      const int rank = __popcll(same & ((uint64_t{1} << lane) - 1));
      const bool last = in && rank + 1 == __popcll(same);
      if (last) seen[wave][r] = static_cast<unsigned short>(rank + 1);
      __syncthreads();
      if (in) {
        int at = next[r] + rank;
        for (int w = 0; w < wave; ++w) at += seen[w][r];
        a.order[at] = Place{list_pos[i], (r << a.group_bits) + mine};
      }
      __syncthreads();
      if (last) {
        atomicAdd(&next[r], rank + 1);
        seen[wave][r] = 0;
      }
      __syncthreads();
    }
  }
}

struct BwdArgs {
  const void* grad;
  void* dw;
  const Segment* segments;
  const Place* order;
  const int* total;
  float* sums;  // [2 * bins][width], see sum_pieces
  int64_t first, count;  // rows of dw, places or pieces of this launch
  int64_t bins;          // of kPiece places
  DivMagic by_pieces;
  int width, pieces;     // pieces of C columns per row
  float scale;
};

// sum[c] += grad[position][col + c] over order[from, to), in order, with
// eight rows' loads in flight.
template <typename T, int C, bool WHOLE>
__device__ __forceinline__ void add_rows(float (&sum)[C], const BwdArgs& a, int from, int to,
                                         int col) {
  constexpr int kFlight = 8;
  const T* grad = static_cast<const T*>(a.grad) + col;
  const int left = a.width - col;
  for (int i0 = from; i0 < to; i0 += kFlight) {
    int64_t at[kFlight];
    Values<T, C> x[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      at[k] = static_cast<int64_t>(a.order[i0 + k < to ? i0 + k : to - 1].position) * a.width;
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      if (WHOLE || left >= C) x[k].load_stream(grad + at[k]);
      else x[k].load_part(grad + at[k], left);
    }
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
#pragma unroll
      for (int c = 0; c < C; ++c) sum[c] += i0 + k < to ? x[k].get(c) : 0.0f;
    }
  }
}

// The sum of each piece of kPiece positions of a token with more than that.
// Pieces are counted from the token's first place s, and the sorted places are
// cut into bins of kPiece: a bin holds the start of at most one piece after a
// token's first (kept in sums[bin]) and of at most one first piece (in
// sums[bins + bin]; its token reaches into the next bin).
template <typename T, int C, bool WHOLE>
__global__ __launch_bounds__(kThreads) void sum_pieces(BwdArgs a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t slot = div_by(id, a.by_pieces);
  if (slot >= a.count) return;
  const int col = static_cast<int>(id - slot * a.pieces) * C;
  const int64_t s = a.first + slot;
  const bool first = s >= a.bins;
  const int bin = static_cast<int>(first ? s - a.bins : s);
  const int total = *a.total;
  const int64_t probe = (static_cast<int64_t>(bin) + (first ? 1 : 0)) * kPiece;
  if (probe >= total) return;
  const Segment g = a.segments[a.order[probe].row];
  if (g.count <= kPiece) return;
  int from;
  if (first) {
    if (g.start < bin * kPiece || g.start >= probe) return;
    from = g.start;
  } else {
    from = g.start + (static_cast<int>(probe) - g.start + kPiece - 1) / kPiece * kPiece;
    if (from == g.start || from >= g.start + g.count) return;
  }
  float sum[C];
#pragma unroll
  for (int c = 0; c < C; ++c) sum[c] = 0.0f;
  add_rows<T, C, WHOLE>(sum, a, from, std::min(from + kPiece, g.start + g.count), col);
  float* to = a.sums + s * a.width + col;
  Values<float, 4> v;
#pragma unroll
  for (int c = 0; c < C; c += 4) {
    const float part[4] = {sum[c], sum[c + 1], sum[c + 2], sum[c + 3]};
    v.set(part);
    const int left = a.width - col - c;
    if (WHOLE || left >= 4) v.store(to + c);
    else if (left > 0) v.store_part(to + c, left);
  }
}

// ADD: rows are those of the places that start a token, added to dw; otherwise
// rows of dw, written.
template <typename T, typename O, int C, bool WHOLE, bool ADD>
__global__ __launch_bounds__(kThreads) void write_rows(BwdArgs a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t r = div_by(id, a.by_pieces);
  if (r >= a.count) return;
  const int col = static_cast<int>(id - r * a.pieces) * C;
  int64_t row = a.first + r;
  if constexpr (ADD) {
    const int64_t place = row;
    if (place >= *a.total) return;
    row = a.order[place].row;
    if (a.segments[row].start != place) return;
  }
  const Segment g = a.segments[row];
  float sum[C];
#pragma unroll
  for (int c = 0; c < C; ++c) sum[c] = 0.0f;
  const int left = a.width - col;
  if (g.count <= kPiece) {
    add_rows<T, C, WHOLE>(sum, a, g.start, g.start + g.count, col);
  } else {
    constexpr int kFlight = 8;
    const int n = (g.count + kPiece - 1) / kPiece;
    for (int j0 = 0; j0 < n; j0 += kFlight) {
      Values<float, 4> x[kFlight][C / 4];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int j = j0 + k < n ? j0 + k : n - 1;
        const int64_t slot = (j == 0 ? a.bins : 0) + (g.start + j * kPiece) / kPiece;
        const float* p = a.sums + slot * a.width + col;
#pragma unroll
        for (int c = 0; c < C; c += 4) {
          if (WHOLE || left >= c + 4) x[k][c / 4].load(p + c);
          else x[k][c / 4].load_part(p + c, left - c);
        }
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
#pragma unroll
        for (int c = 0; c < C; ++c) sum[c] += j0 + k < n ? x[k][c / 4].get(c % 4) : 0.0f;
      }
    }
  }
  O* dw = static_cast<O*>(a.dw) + row * a.width + col;
  Values<O, C> v;
  if constexpr (ADD) {
    if (WHOLE || left >= C) v.load(dw);
    else v.load_part(dw, left);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) sum[c] = ADD ? v.get(c) + sum[c] * a.scale : sum[c] * a.scale;
  v.set(sum);
  if (WHOLE || left >= C) v.store_stream(dw);
  else v.store_part(dw, left);
}

// Workspace: the order, the rows' segments, the number of places, the sums of
// pieces; each 16-byte aligned.
struct Layout {
  int64_t bins;
  size_t segments, total, sums, bytes;
};

inline Layout layout(int64_t count, int64_t width, int64_t vocab) {
  const auto up = [](size_t n) { return (n + 15) / 16 * 16; };
  Layout l;
  l.bins = (count + kPiece - 1) / kPiece;
  l.segments = up(count * sizeof(Place));
  l.total = l.segments + up(vocab * sizeof(Segment));
  l.sums = l.total + 16;
  // A token with more than kPiece places needs that many.
  l.bytes = l.sums + (count > kPiece ? 2 * l.bins * width * sizeof(float) : 0);
  return l;
}

// LAUNCH(first, count, blocks) over `rows` rows of `pieces` lanes each.
template <typename F>
void for_lanes(int64_t rows, int64_t pieces, F&& launch) {
  const int64_t step = std::max<int64_t>(1, kLanes / pieces);
  for (int64_t first = 0; first < rows; first += step) {
    const int64_t n = std::min(step, rows - first);
    launch(first, n, dim3(static_cast<unsigned>((n * pieces + kThreads - 1) / kThreads)));
  }
}

template <typename T, typename O>
void launch_bwd(BwdArgs a, const SortArgs& s, bool accumulate, hipStream_t stream) {
  constexpr int C = 16 / std::max(sizeof(T), sizeof(O));
  const bool whole = a.width % C == 0;
  a.pieces = (a.width + C - 1) / C;
  a.by_pieces = div_magic(a.pieces);
  if (s.count > 0 || !accumulate) {
    sort_tokens<<<dim3(1u << s.group_bits), dim3(kSortThreads), 0, stream>>>(s);
  }
  const auto run = [&](auto kernel, int64_t rows) {
    for_lanes(rows, a.pieces, [&](int64_t first, int64_t n, dim3 grid) {
      a.first = first;
      a.count = n;
      kernel<<<grid, dim3(kThreads), 0, stream>>>(a);
    });
  };
  if (s.count > kPiece) {
    run(whole ? sum_pieces<T, C, true> : sum_pieces<T, C, false>, 2 * a.bins);
  }
  if (accumulate) {
    run(whole ? write_rows<T, O, C, true, true> : write_rows<T, O, C, false, true>, s.count);
  } else {
    run(whole ? write_rows<T, O, C, true, false> : write_rows<T, O, C, false, false>, s.vocab);
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
  const int c = 16 / elem_size;
  const bool whole = width % c == 0;
  const int pieces = static_cast<int>((width + c - 1) / c);
  FwdArgs a{weight, tokens, out, 0, 0, vocab, row_stride, div_magic(pieces),
            static_cast<int>(width), pieces, scale, token_size};
  auto kernel = elem_size == 2
                    ? (whole ? embedding_rows<uint16_t, true> : embedding_rows<uint16_t, false>)
                    : (whole ? embedding_rows<float, true> : embedding_rows<float, false>);
  for_lanes(count, pieces, [&](int64_t first, int64_t n, dim3 grid) {
    a.first = first;
    a.count = n;
    kernel<<<grid, dim3(kThreads), 0, stream>>>(a);
  });
  return check_launch("embedding");
}

extern "C" size_t hipo_embedding_bwd_workspace_bytes(int64_t count, int64_t width,
                                                     int64_t vocab) {
  if (count < 0 || width <= 0 || vocab <= 0) return 0;
  return hipo::layout(count, width, vocab).bytes;
}

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
  HIPO_REQUIRE(count <= 0x7fffffff - kPiece && width <= 0x7fffffff && vocab <= 0x7fffffff,
               "embedding_bwd: size over 2^31");
  if (width == 0 || vocab == 0) return 0;
  HIPO_REQUIRE(dweight != nullptr && (count == 0 || (grad != nullptr && tokens != nullptr)),
               "embedding_bwd: null pointer");
  const Layout l = layout(count, width, vocab);
  HIPO_REQUIRE(workspace != nullptr && workspace_bytes >= l.bytes,
               "embedding_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, l.bytes);
  HIPO_REQUIRE(aligned16(workspace), "embedding_bwd: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  BwdArgs a{};
  a.grad = grad;
  a.dw = dweight;
  a.order = reinterpret_cast<Place*>(ws);
  a.segments = reinterpret_cast<Segment*>(ws + l.segments);
  a.total = reinterpret_cast<int*>(ws + l.total);
  a.sums = reinterpret_cast<float*>(ws + l.sums);
  a.bins = l.bins;
  a.width = static_cast<int>(width);
  a.scale = scale;
  SortArgs s{tokens, reinterpret_cast<Segment*>(ws + l.segments), reinterpret_cast<Place*>(ws),
             reinterpret_cast<int*>(ws + l.total), count, vocab, padding_idx, token_size, 0};
  while ((int64_t{1} << s.group_bits) < kSortGroups ||
         (int64_t{kSortRows} << s.group_bits) < vocab) {
    ++s.group_bits;
  }
  if (elem_size == 2) {
    if (out_size == 2) launch_bwd<uint16_t, uint16_t>(a, s, accumulate != 0, stream);
    else launch_bwd<uint16_t, float>(a, s, accumulate != 0, stream);
  } else {
    if (out_size == 2) launch_bwd<float, uint16_t>(a, s, accumulate != 0, stream);
    else launch_bwd<float, float>(a, s, accumulate != 0, stream);
  }
  return check_launch("embedding_bwd");
}
