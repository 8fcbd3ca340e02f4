// Embedding lookup with a scale, and its gradient:
//   out[t] = scale * w[token_t],    dw[v] = scale * sum_{t: token_t = v} grad[t],
// the sum in fp32 in an order that the tokens alone fix, one rounding at the
// end.  Both move rows: HBM bounds them.
//
// Lookup: a lane per 16-byte piece of the output, pieces in memory order, so
// no lane is idle whatever the width.  Non-temporal stores (cached ones: 1.6
// times as long); [8192, 4096] bf16 16.4 us, 6.0 TB/s.  Each XCD writes an eighth
// of the output, so that lines that two rows share are merged in one L2: us, by
// XCD / in the launch's order, [20011, 1001] fp32 19.0 / 20.4, [20011, 2001] bf16
// 21.0 / 22.7, [20011, 1000] fp32 18.1 / 18.7; where rows share no line it gains
// nothing, [8192, 4096] bf16 16.4 / 16.0, and one order serves all widths.  In
// the launch's order two / four pieces per lane took 17.2 / 17.5 there, pieces
// aligned in the output 21.4 at [20011, 1001].
//
// Gradient, three launches:
//   1. sort_tokens: the positions in order of their token, equal tokens in
//      order of position.  A workgroup owns the tokens with one remainder
//      modulo the number of workgroups (a vocabulary is ordered by frequency:
//      ranges of it would give one workgroup most of the tokens) and scans all
//      tokens, counting the smaller remainders on the way: no exchange between
//      workgroups, no atomics on memory.  Arithmetic bounds the scan, about
//      200 cycles per 64 tokens and SIMD: 6.6 us at 8192 tokens, 21 us at
//      65536.  A workgroup holds 512 rows: from 65536 rows on there are vocab / 512
//      of them, and each scans all tokens.  All three launches, 2048 / 65536 tokens
//      of width 8 added into 65536 rows 12 / 23 us, 200000 13 / 31, 10^6 26 / 79, 10^7
//      262 / 972, 10^8 2030 / 7630.
//      Other workgroups of the same launch write zeros to all of dw: most of
//      the bytes where tokens are fewer than rows ([128000, 4096] bf16 158 us,
//      6.6 TB/s), and beside the sort hardly any time where they are not (rows
//      without a token found and zeroed by sum_rows instead: [65536, 2048] into
//      [32000, 2048] 106.5 us against 101.4, [65536, 64] into [1696, 64] 38.2
//      against 39.1).
//   2. sum_rows: a lane per 16 bytes of a gradient row's columns and place that
//      starts a token: the sum of its few positions.  Tokens that occur more
//      often than a piece is long are cut into pieces, summed in the same
//      launch into the workspace (fp32);
//   3. join_pieces: their rows, the sums of their pieces.
// Few tokens take one launch instead, sum_few.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "hipo_common.h"

namespace hipo {
namespace {

constexpr int kThreads = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortLoads = 8;        // tokens per thread in flight
constexpr int kSortList = 512;       // tokens a sorting wave keeps
constexpr int kSortRows = 512;       // rows of dw per sorting workgroup
constexpr int kSortRowBits = 9;
constexpr int64_t kSortPart = int64_t{1} << (32 - kSortRowBits);  // positions a list can tell
// At least: the other half of the CUs writes zeros (256: [2048, 768] into [32000,
// 768] 20.1 us instead of 19.1, [65536, 2048] into [32000, 2048] 104.7 instead of
// 101.1; nothing else within 2 %).
constexpr int kSortGroups = 128;
constexpr int kFewTokens = 1024;     // summed without a sort
constexpr int kFewThreads = 512;
constexpr int kFewFill = 2;          // zeros: 16-byte pieces per thread
constexpr int64_t kLanes = int64_t{1} << 30;  // lanes per launch
// A launch has fewer than 2^32 threads, fewer than 2^22 workgroups of 1024: 2^21 sort
// where there are 2^30 rows; of the others as many as are left and 8 XCDs can share.
constexpr int64_t kFillBlocks = (int64_t{1} << 21) - 8;

__device__ __forceinline__ int64_t token_at(const void* tokens, int size, int64_t i) {
  return size == 8 ? static_cast<const int64_t*>(tokens)[i]
                   : static_cast<const int32_t*>(tokens)[i];
}

// C consecutive values at any element alignment, as they lie in memory.
template <typename T, int C>
struct Values {
  typedef T Vec __attribute__((ext_vector_type(C)));
  typedef Vec Unaligned __attribute__((aligned(sizeof(T))));
  Vec v;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = T{0};
  }
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
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x) * kThreads + threadIdx.x;
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

// A token's places in the sorted order.
struct Segment {
  int start, count;
};
struct Place {
  int position, row;
  Segment token;  // all places of this row
};

struct SortArgs {
  const void* tokens;
  Place* order;       // [count]
  int* total;         // tokens that count
  uint16_t* fill;     // zeroed by the workgroups after the sorting ones
  int64_t fill_values;
  int64_t count, vocab, padding_idx;
  int group_bits;     // 2^group_bits sorting workgroups
};

// Zeros, 16 bytes per thread (64: [128000, 4096] bf16 221 us instead of 173);
// more where dw is over kFillBlocks * 16 KiB.  Each XCD writes an eighth of dw:
// 8192 tokens into [128000, 4096] 183.7 us in all instead of 204.4, 4096 into
// [50000, 2048] fp32 76.9 instead of 81.4.
__device__ __forceinline__ void fill_zeros(const SortArgs& a, uint32_t block, uint32_t blocks) {
  Values<uint16_t, 8> zero;
  zero.clear();
  const int64_t first = int64_t{xcd_order(block, blocks)} * kSortThreads + threadIdx.x;
  for (int64_t at = first * 8; at < a.fill_values; at += int64_t{blocks} * kSortThreads * 8) {
    if (at + 8 <= a.fill_values) zero.store_stream(a.fill + at);
    else zero.store_part(a.fill + at, static_cast<int>(a.fill_values - at));
  }
}

// kSortLoads tokens of a lane, 64 positions apart from `at` (of the wave) on;
// past the end the last one.
template <typename I>
__device__ __forceinline__ void load_tokens(const SortArgs& a, int64_t at, I (&v)[kSortLoads]) {
  const I* p = static_cast<const I*>(a.tokens) + at;
  const int lane = threadIdx.x & (kWave - 1);
  if (at + kSortLoads * kWave <= a.count) {
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) v[u] = p[lane + u * kWave];
  } else {
    const int last = static_cast<int>(a.count - 1 - at);
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) v[u] = p[std::min(lane + u * kWave, last)];
  }
  __builtin_amdgcn_sched_barrier(0);  // the loads first
}

// A wave's next places of the rows, one row per lane (-1: none), lanes in
// order: stable.
__device__ __forceinline__ int take_places(int r, int* next, bool& last) {
  uint64_t same = __ballot(r >= 0);
#pragma unroll
  for (int b = 0; b < kSortRowBits; ++b) {
    const uint64_t m = __ballot((r >> b) & 1);
    same &= ((r >> b) & 1) ? m : ~m;
  }
  const int rank = __popcll(same & ((uint64_t{1} << (threadIdx.x & (kWave - 1))) - 1));
  const int place = r >= 0 ? next[r] + rank : 0;
  last = r >= 0 && rank + 1 == __popcll(same);
  return place;
}

// The waves of a workgroup take consecutive parts of the tokens, in order, so
// that each has its own counts and places and none waits for another but
// between the count and the places.  A wave keeps what it finds in a list in
// LDS; one that finds more than the list holds reads its part again.
template <typename I>
__global__ __launch_bounds__(kSortThreads, 8) void sort_tokens(SortArgs a) {
  __shared__ int found[kSortWaves][kSortRows];  // counts, then next places
  __shared__ Segment token[kSortRows];
  __shared__ uint32_t list[kSortWaves][kSortList];  // place in the part, row
  __shared__ int wave_count[kSortWaves];
  __shared__ int wave_below[kSortWaves];
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = 1 << a.group_bits;
  const int mine = blockIdx.x;
  if (mine >= groups) {
    fill_zeros(a, mine - groups, gridDim.x - groups);
    return;
  }
  const int64_t part = (a.count + kSortThreads - 1) / kSortThreads * kWave;  // of a wave
  const int64_t from = wave * part;
  const int64_t to = from + part < a.count ? from + part : a.count;
  constexpr int kBatch = kSortLoads * kWave;
  I v[2][kSortLoads];  // a batch and the one after it
  if (from < to) load_tokens(a, from, v[0]);
  for (int i = tid; i < kSortWaves * kSortRows / 4; i += kSortThreads)
    reinterpret_cast<u32x4_t*>(&found[0][0])[i] = u32x4_t{0u, 0u, 0u, 0u};
  __syncthreads();

  // A token that counts is a 32-bit number; what it leaves modulo the number
  // of groups, or no group's number.
  const uint32_t vocab = static_cast<uint32_t>(a.vocab);
  const uint32_t padding = a.padding_idx >= 0 && a.padding_idx < a.vocab
                               ? static_cast<uint32_t>(a.padding_idx)
                               : 0xffffffffu;
  const uint32_t mask = static_cast<uint32_t>(groups) - 1;
  const auto group_of = [&](I x, bool in) -> uint32_t {
    const uint32_t t = static_cast<uint32_t>(x);
    bool counts = in && t < vocab && t != padding;
    if constexpr (sizeof(I) == 8) counts = counts && static_cast<uint64_t>(x) >> 32 == 0;
    return counts ? t & mask : 0xffffffffu;
  };
  const auto row_of = [&](I x) { return static_cast<int>(static_cast<uint32_t>(x) >> a.group_bits); };

  int below = 0, held = 0;  // of the wave
  const auto scan = [&](auto whole, const I (&x)[kSortLoads], int64_t i0) {
    const int left = static_cast<int>(std::min<int64_t>(to - i0, kBatch));
    const uint32_t part_at = static_cast<uint32_t>(i0 - from) + lane;
#pragma unroll
    for (int u = 0; u < kSortLoads; ++u) {
      const uint32_t g = group_of(x[u], whole || u * kWave + lane < left);
      below += __popcll(__ballot(g < static_cast<uint32_t>(mine)));
      const bool own = g == static_cast<uint32_t>(mine);
      const uint64_t m = __ballot(own);
      if (m == 0) continue;
      const int slot = held + __popcll(m & ((uint64_t{1} << lane) - 1));
      if (own) {
        const int r = row_of(x[u]);
        atomicAdd(&found[wave][r], 1);
        if (slot < kSortList) list[wave][slot] = (part_at + u * kWave) << kSortRowBits | r;
      }
      held += __popcll(m);
    }
  };
  const auto scan_batch = [&](const I (&x)[kSortLoads], int64_t i0) {
    if (i0 + kBatch <= to) scan(std::true_type{}, x, i0);
    else scan(std::false_type{}, x, i0);
  };
  for (int64_t i0 = from; i0 < to; i0 += 2 * kBatch) {
    if (i0 + kBatch < to) load_tokens(a, i0 + kBatch, v[1]);
    scan_batch(v[0], i0);
    if (i0 + kBatch >= to) break;
    if (i0 + 2 * kBatch < to) load_tokens(a, i0 + 2 * kBatch, v[0]);
    scan_batch(v[1], i0 + kBatch);
  }
  if (lane == 0) wave_below[wave] = below;
  __syncthreads();

  // Exclusive sums over the rows, one row per thread, then over the waves.
  int n = 0;
  if (tid < kSortRows) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) n += found[w][tid];
  }
  int sum = n;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == kWave - 1) wave_count[wave] = sum;
  __syncthreads();
  int start = sum - n;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    start += wave_below[w];
    if (w < wave) start += wave_count[w];
  }
  if (tid < kSortRows) {
    const Segment g{start, n};
    token[tid] = g;
    int next = start;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = found[w][tid];
      found[w][tid] = next;
      next += c;
    }
    if (mine == groups - 1 && tid == kSortRows - 1) *a.total = start + n;
  }
  __syncthreads();

  const auto write = [&](int r, int64_t at) {
    bool last;
    const int place = take_places(r, found[wave], last);
    if (r >= 0) {
      a.order[place] = Place{static_cast<int>(at), (r << a.group_bits) + mine, token[r]};
      if (last) found[wave][r] = place + 1;
    }
    __builtin_amdgcn_wave_barrier();  // the wave's other lanes read it next
  };
  if (held <= kSortList && part <= kSortPart) {
    for (int l0 = 0; l0 < held; l0 += kWave) {
      const bool in = l0 + lane < held;
      const uint32_t e = in ? list[wave][l0 + lane] : 0;
      write(in ? static_cast<int>(e & (kSortRows - 1)) : -1, from + (e >> kSortRowBits));
    }
  } else {
    for (int64_t i0 = from; i0 < to; i0 += kBatch) {
      load_tokens(a, i0, v[0]);
      const int left = static_cast<int>(std::min<int64_t>(to - i0, kBatch));
#pragma unroll 1
      for (int u = 0; u < kSortLoads; ++u) {
        I x = v[0][0];  // v[0][u], kept in registers
#pragma unroll
        for (int k = 1; k < kSortLoads; ++k) x = u == k ? v[0][k] : x;
        const uint32_t g = group_of(x, u * kWave + lane < left);
        write(g == static_cast<uint32_t>(mine) ? row_of(x) : -1, i0 + u * kWave + lane);
      }
    }
  }
}

struct BwdArgs {
  const void* grad;
  void* dw;
  const Place* order;
  const int* total;
  float* sums;           // [2 * bins][width], see first_piece
  int64_t first, count;  // slots of this launch
  int64_t places;        // in order, of which *total are filled
  int64_t bins;          // of 2^bits places
  int bits;              // of a piece
  DivMagic by_pieces;
  int width, pieces;     // pieces of C columns per row
  float scale;
};

// sum[c] += grad[position][col + c] over order[from, to), in order, with
// FLIGHT rows' loads in flight.  sum_rows with 4 / 8 / 16, us: [2048, 768] into
// [32000, 768] 10.9 / 7.8 / 6.5, [8192, 4096] into [128000, 4096] 23.6 / 23.1 /
// 28.0, [16381, 2880] added into fp32 [50001, 2880] 39.6 / 39.2 / 45.4.
template <typename T, int C, bool WHOLE, int FLIGHT>
__device__ __forceinline__ void add_rows(float (&sum)[C], const BwdArgs& a, int from, int to,
                                         int col) {
  const T* grad = static_cast<const T*>(a.grad) + col;
  const int left = a.width - col;
  for (int i0 = from; i0 < to; i0 += FLIGHT) {
    // The barriers: or the compiler waits for each load before it issues the
    // next.  No load where there is no row: most tokens occur once or twice.
    int at[FLIGHT];
    Values<T, C> x[FLIGHT];
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) {
      at[k] = 0;
      if (i0 + k < to) at[k] = a.order[i0 + k].position;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) {
      x[k].clear();
      if (i0 + k < to) {
        const T* p = grad + static_cast<int64_t>(at[k]) * a.width;
        if (WHOLE || left >= C) x[k].load_stream(p);
        else x[k].load_part(p, left);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < FLIGHT; ++k) {
#pragma unroll
      for (int c = 0; c < C; ++c) sum[c] += x[k].get(c);
    }
  }
}

// Tokens with more than 2^bits places are summed in pieces of that many,
// counted from the token's first place.  The sorted places are cut into bins
// of the same size: a bin holds the start of at most one piece after a token's
// first (its sum is kept in sums[bin]) and of at most one first piece (in
// sums[bins + bin]; its token reaches into the next bin).
__device__ __forceinline__ bool in_pieces(const BwdArgs& a, Segment token) {
  return token.count > 1 << a.bits;
}

// The token of a bin's first piece, count 0 if there is none.
__device__ __forceinline__ Segment first_piece(const BwdArgs& a, int bin) {
  const int64_t probe = (int64_t{bin} + 1) << a.bits;
  const int total = *a.total;
  const Segment g = a.order[probe < a.places ? probe : a.places - 1].token;
  const bool here = probe < total && in_pieces(a, g) && g.start < probe &&
                    g.start >= probe - (1 << a.bits);
  return here ? g : Segment{0, 0};
}

// The places of slot's piece, from == to if there is none.
__device__ __forceinline__ void piece_places(const BwdArgs& a, int64_t slot, int& from, int& to) {
  const int size = 1 << a.bits;
  from = to = 0;
  Segment g;
  if (slot >= a.bins) {
    g = first_piece(a, static_cast<int>(slot - a.bins));
    if (g.count == 0) return;
    from = g.start;
  } else {
    const int64_t probe = slot << a.bits;
    const int total = *a.total;
    g = a.order[probe].token;
    if (probe >= total || !in_pieces(a, g)) return;
    const int at = g.start + ((static_cast<int>(probe) - g.start + size - 1) & -size);
    if (at == g.start || at >= g.start + g.count) return;
    from = at;
  }
  to = std::min(from + size, g.start + g.count);
}

// A lane's C columns of a row of dw.
template <typename O, int C, bool WHOLE, bool ADD>
struct Row {
  O* dw;
  int left;
  Values<O, C> had;

  // What is there is loaded at once: beside the gradient rows, not after them.
  __device__ __forceinline__ Row(const BwdArgs& a, int64_t row, int col)
      : dw(static_cast<O*>(a.dw) + row * a.width + col), left(a.width - col) {
    if constexpr (ADD) {
      if (WHOLE || left >= C) had.load(dw);
      else had.load_part(dw, left);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __device__ __forceinline__ void write(float (&sum)[C], float scale) {
#pragma unroll
    for (int c = 0; c < C; ++c) sum[c] = ADD ? had.get(c) + sum[c] * scale : sum[c] * scale;
    had.set(sum);
    if (WHOLE || left >= C) had.store_stream(dw);
    else had.store_part(dw, left);
  }
};

// A lane per C columns of a piece (the first 2 * bins slots) or of a place:
// one that starts a token sums and writes its row.  Tokens in pieces are left
// to join_pieces; rows without a token are zeros already, or stay.  ADD: added
// to dw.
template <typename T, typename O, int C, bool WHOLE, bool ADD>
__global__ __launch_bounds__(kThreads) void sum_rows(BwdArgs a) {
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t r = div_by(id, a.by_pieces);
  if (r >= a.count) return;
  const int col = static_cast<int>(id - r * a.pieces) * C;
  const int left = a.width - col;
  const int64_t slot = a.first + r;
  float sum[C] = {};
  if (slot < 2 * a.bins) {
    int from, to;
    piece_places(a, slot, from, to);
    if (from == to) return;
    add_rows<T, C, WHOLE, 8>(sum, a, from, to, col);
    float* p = a.sums + slot * a.width + col;
    Values<float, C> v;
    v.set(sum);
    if (WHOLE || left >= C) v.store(p);
    else v.store_part(p, left);
    return;
  }
  const int64_t place = slot - 2 * a.bins;
  const int total = *a.total;
  // One load for all of it, beside the total's.
  const Place p = __builtin_bit_cast(Place, *reinterpret_cast<const u32x4_t*>(a.order + place));
  const Segment g = p.token;
  if (place >= total || g.start != place || in_pieces(a, g)) return;
  // Its first position is in hand.
  const T* grad = static_cast<const T*>(a.grad) + int64_t{p.position} * a.width + col;
  Values<T, C> x;
  if (WHOLE || left >= C) x.load_stream(grad);
  else x.load_part(grad, left);
  Row<O, C, WHOLE, ADD> out(a, p.row, col);
#pragma unroll
  for (int c = 0; c < C; ++c) sum[c] += x.get(c);
  add_rows<T, C, WHOLE, 8>(sum, a, g.start + 1, g.start + g.count, col);
  out.write(sum, a.scale);
}

// The rows of tokens in pieces: a workgroup per bin and 64 lanes of C columns
// each, its waves a quarter of the pieces each, added in order.
template <typename O, int C, bool WHOLE, bool ADD>
__global__ __launch_bounds__(kThreads) void join_pieces(BwdArgs a) {
  constexpr int kWaves = kThreads / kWave, kFlight = 8;
  __shared__ float part[kWaves][C][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const uint32_t r = div_by(blockIdx.x, a.by_pieces);
  const int col = (static_cast<int>(blockIdx.x - r * a.pieces) * kWave + lane) * C;
  const int left = a.width - col;
  const int bin = static_cast<int>(a.first + r);
  const Segment g = first_piece(a, bin);
  if (g.count == 0) return;  // the whole workgroup
  const int row = a.order[g.start].row;
  const float* sums = a.sums + col;
  const int n = (g.count + (1 << a.bits) - 1) >> a.bits;
  const int each = (n + kWaves - 1) / kWaves;
  const int to = std::min(n, (wave + 1) * each);
  float sum[C] = {};
  if (left > 0) {
    for (int j0 = wave * each; j0 < to; j0 += kFlight) {
      Values<float, C> x[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        x[k].clear();
        const int j = j0 + k;
        if (j < to) {
          const float* p = sums + ((j == 0 ? a.bins : 0) + int64_t{bin} + j) * a.width;
          if (WHOLE || left >= C) x[k].load(p);
          else x[k].load_part(p, left);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
#pragma unroll
        for (int c = 0; c < C; ++c) sum[c] += x[k].get(c);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) part[wave][c][lane] = sum[c];
  __syncthreads();
  if (wave != 0 || left <= 0) return;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
#pragma unroll
    for (int c = 0; c < C; ++c) sum[c] += part[w][c][lane];
  }
  Row<O, C, WHOLE, ADD>(a, row, col).write(sum, a.scale);
}

// ---------------------------------------------------------------------------
// Few tokens: no sort.  A workgroup per position and 64 lanes' columns looks
// through all tokens: where its own occurs first it sums all of that token's
// rows, each wave a part of them.  Workgroups behind those write the zeros of
// the other rows (a launch of zeros before it: [17, 94] fp32 into 13054 rows
// 6.7 us instead of 5.0, [16, 2880] into [50001, 2880] fp32 100.8 instead of 92.1).
// ---------------------------------------------------------------------------

struct FewArgs {
  const void* grad;
  const void* tokens;
  void* dw;
  int64_t vocab, padding_idx;
  DivMagic by_chunks, by_width;
  int count, width, chunks;  // workgroups per row
  float scale;
  int token_size;
};

// Zeros to kFewFill 16-byte pieces of dw per thread, but not to rows that a
// token takes: those are marked first.  Each XCD writes an eighth of dw: 64
// tokens into [128000, 4096] bf16 165.6 us instead of 179.2, 128 into [32000, 768]
// 11.8 instead of 11.5.  With one / two / four pieces 200.1 / 165.6 / 177.5 and
// 15.2 / 11.8 / 11.9.
template <typename O>
__device__ __forceinline__ void zero_other_rows(const FewArgs& f, int64_t block, uint32_t* marks) {
  constexpr int C = 16 / sizeof(O), kValues = kFewThreads * kFewFill * C;
  static_assert(kValues <= kFewTokens * 32);
  const int tid = threadIdx.x;
  const int64_t from = block * kValues;
  const int values = static_cast<int>(std::min<int64_t>(f.vocab * f.width - from, kValues));
  const int64_t row0 = from / f.width;
  const int skip = static_cast<int>(from - row0 * f.width);
  const int rows = static_cast<int>(div_by(skip + values - 1, f.by_width)) + 1;
  int64_t mine[kFewTokens / kFewThreads];
#pragma unroll
  for (int k = 0; k < kFewTokens / kFewThreads; ++k) {
    const int i = k * kFewThreads + tid;
    mine[k] = i < f.count ? token_at(f.tokens, f.token_size, i) : -1;
  }
  for (int i = tid; i < (rows + 31) / 32; i += kFewThreads) marks[i] = 0;
  __syncthreads();
  int taken = 0;
#pragma unroll
  for (int k = 0; k < kFewTokens / kFewThreads; ++k) {
    if (mine[k] >= row0 && mine[k] < row0 + rows && mine[k] != f.padding_idx) {
      const uint32_t r = static_cast<uint32_t>(mine[k] - row0);
      atomicOr(marks + r / 32, 1u << (r % 32));
      taken = 1;
    }
  }
  taken = __syncthreads_or(taken);
  O* dw = static_cast<O*>(f.dw) + from;
  Values<O, C> zero;
  zero.clear();
  const auto marked = [&](int v) {
    const uint32_t r = div_by(skip + v, f.by_width);
    return (marks[r / 32] >> (r % 32)) & 1;
  };
#pragma unroll
  for (int k = 0; k < kFewFill; ++k) {
    const int v = (k * kFewThreads + tid) * C;
    if (v >= values) break;
    const int n = std::min(values - v, C);
    if (!taken || (f.width >= C && !marked(v) && !marked(v + n - 1))) {
      if (n == C) zero.store_stream(dw + v);
      else zero.store_part(dw + v, n);
    } else {
      for (int c = 0; c < n; ++c) {
        if (!marked(v + c)) dw[v + c] = O{0};
      }
    }
  }
}

template <typename T, typename O, int C, bool WHOLE, bool ADD>
__global__ __launch_bounds__(kFewThreads) void sum_few(FewArgs f) {
  constexpr int kWaves = kFewThreads / kWave, kLooks = kFewTokens / kFewThreads, kFlight = 8;
  __shared__ uint64_t same[kLooks * kWaves];  // of each 64 positions
  __shared__ int list[kFewTokens];
  __shared__ float part[kWaves][C][kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  if (!ADD && blockIdx.x >= static_cast<unsigned>(f.count * f.chunks)) {
    const uint32_t sums = f.count * f.chunks;
    zero_other_rows<O>(f, xcd_order(blockIdx.x - sums, gridDim.x - sums),
                       reinterpret_cast<uint32_t*>(list));
    return;
  }
  const int t = static_cast<int>(div_by(blockIdx.x, f.by_chunks));
  const int col = ((static_cast<int>(blockIdx.x) - t * f.chunks) * kWave + lane) * C;
  const int64_t token = token_at(f.tokens, f.token_size, t);
  uint64_t m[kLooks];
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    const int i = k * kFewThreads + tid;
    m[k] = __ballot(i < f.count && token_at(f.tokens, f.token_size, i) == token);
    if (lane == 0) same[k * kWaves + wave] = m[k];
  }
  if (token < 0 || token >= f.vocab || token == f.padding_idx) return;  // the workgroup
  __syncthreads();
  int n = 0, first = f.count, before[kLooks];
#pragma unroll
  for (int j = 0; j < kLooks * kWaves; ++j) {
    const uint64_t b = same[j];
    if (j % kWaves == wave) before[j / kWaves] = n;
    if (n == 0 && b != 0) first = j * kWave + __builtin_ctzll(b);
    n += __popcll(b);
  }
  if (first != t) return;  // the workgroup
#pragma unroll
  for (int k = 0; k < kLooks; ++k) {
    if ((m[k] >> lane) & 1)
      list[before[k] + __popcll(m[k] & ((uint64_t{1} << lane) - 1))] = k * kFewThreads + tid;
  }
  __syncthreads();
  BwdArgs a{};
  a.dw = f.dw;
  a.width = f.width;
  const bool columns = col < f.width;
  const int left = f.width - col;
  const int each = (n + kWaves - 1) / kWaves;
  const int to = std::min(n, (wave + 1) * each);
  float sum[C] = {};
  if (columns) {
    const T* grad = static_cast<const T*>(f.grad) + col;
    for (int i0 = wave * each; i0 < to; i0 += kFlight) {
      Values<T, C> x[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        x[k].clear();
        if (i0 + k < to) {
          const T* p = grad + int64_t{list[i0 + k]} * f.width;
          if (WHOLE || left >= C) x[k].load_stream(p);
          else x[k].load_part(p, left);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
#pragma unroll
        for (int c = 0; c < C; ++c) sum[c] += x[k].get(c);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) part[wave][c][lane] = sum[c];
  __syncthreads();
  if (wave != 0 || !columns) return;
  Row<O, C, WHOLE, ADD> out(a, token, col);
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
#pragma unroll
    for (int c = 0; c < C; ++c) sum[c] += part[w][c][lane];
  }
  out.write(sum, f.scale);
}

// Up to so many tokens and gradient values there is no sort: one launch and no
// workspace.  Graph replays of bf16, us, with the sort / this: added [128, 768] 9.0 /
// 4.7, [512, 512] 11.0 / 5.6, [1024, 64] 13.1 / 7.4, [1024, 768] 12.6 / 11.4; of one
// token alone 10.5 / 5.4, 11.4 / 9.8, 13.3 / 16.1, 14.0 / 20.2.  [512, 512] with 256
// threads 5.0 and 14.9, with 1024 7.1 and 9.4.
// 2^31 threads write the zeros of 2^34 fp32 values.
inline bool few_tokens(int64_t count, int64_t width, int64_t vocab) {
  return count <= kFewTokens && width <= (1 << 19) / std::max<int64_t>(count, 1) &&
         vocab <= (int64_t{1} << 34) / width;
}

// Workspace: the order, the number of places, the sums of pieces; each 16-byte
// aligned.
struct Layout {
  int bits;
  int64_t bins;
  size_t total, sums, bytes;
};

inline Layout layout(int64_t count, int64_t width) {
  const auto up = [](size_t n) { return (n + 15) / 16 * 16; };
  Layout l;
  // A piece is as long a chain of loads as the whole call waits for where there
  // is little to read: 8 / 16 / 32 places, us: [2048, 768] into [32000, 768] 16.5
  // / 17.5 / 19.4, [16384, 512] added into [32000, 512] 24.1 / 22.7 / 23.9,
  // [8192, 2048] 26.2 / 26.1 / 26.2, [65536, 2048] into [32000, 2048] 121 / 108 /
  // 102, [65536, 64] into [1696, 64] 55 / 43 / 40.
  l.bits = count <= 32768 && count * width <= 1 << 24 ? 4 : 5;
  l.bins = (count + (1 << l.bits) - 1) >> l.bits;
  l.total = up(count * sizeof(Place));
  l.sums = l.total + 16;
  // A token with more places than a piece needs that many.
  if (count <= 1 << l.bits) l.bins = 0;
  l.bytes = l.sums + 2 * l.bins * width * sizeof(float);
  return l;
}

// launch(first, count, blocks) over `rows` rows of `pieces` lanes each.
template <typename F>
void for_lanes(int64_t rows, int64_t pieces, F&& launch) {
  const int64_t step = std::max<int64_t>(1, kLanes / pieces);
  for (int64_t first = 0; first < rows; first += step) {
    const int64_t n = std::min(step, rows - first);
    launch(first, n, dim3(static_cast<unsigned>((n * pieces + kThreads - 1) / kThreads)));
  }
}

template <typename T, typename O>
int launch_few(const BwdArgs& a, const SortArgs& s, int token_size, bool accumulate,
               hipStream_t stream) {
  constexpr int C = 16 / sizeof(T);
  const bool whole = a.width % C == 0;
  const int chunks = (a.width + C * kWave - 1) / (C * kWave);
  const FewArgs f{a.grad, s.tokens, a.dw, s.vocab, s.padding_idx, div_magic(chunks),
                  div_magic(a.width), static_cast<int>(s.count), a.width, chunks, a.scale,
                  token_size};
  constexpr int64_t kFill = int64_t{kFewThreads} * kFewFill * 16 / sizeof(O);
  const int64_t fills = accumulate ? 0 : (s.vocab * a.width + kFill - 1) / kFill;
  const int64_t groups = f.count * chunks + fills;
  if (groups == 0) return 0;
  auto kernel = accumulate
                    ? (whole ? sum_few<T, O, C, true, true> : sum_few<T, O, C, false, true>)
                    : (whole ? sum_few<T, O, C, true, false> : sum_few<T, O, C, false, false>);
  kernel<<<dim3(static_cast<unsigned>(groups)), dim3(kFewThreads), 0, stream>>>(f);
  return check_launch("embedding_bwd");
}

// Each launch reads what the one before it wrote: none follows one that was refused.
template <typename T, typename O>
int launch_bwd(BwdArgs a, SortArgs s, int token_size, bool accumulate, hipStream_t stream) {
  constexpr int C = 16 / sizeof(T);
  const bool whole = a.width % C == 0;
  a.pieces = (a.width + C - 1) / C;
  a.by_pieces = div_magic(a.pieces);
  auto sort = token_size == 8 ? sort_tokens<int64_t> : sort_tokens<int32_t>;
  constexpr int64_t kPerBlock = int64_t{kSortThreads} * 8;
  const int64_t fill =
      accumulate ? 0 : std::min((s.fill_values + kPerBlock - 1) / kPerBlock, kFillBlocks);
  sort<<<dim3(static_cast<unsigned>((int64_t{1} << s.group_bits) + fill)), dim3(kSortThreads), 0,
         stream>>>(s);
  if (const int rc = check_launch("embedding_bwd")) return rc;
  a.places = s.count;
  auto rows = accumulate
                  ? (whole ? sum_rows<T, O, C, true, true> : sum_rows<T, O, C, false, true>)
                  : (whole ? sum_rows<T, O, C, true, false> : sum_rows<T, O, C, false, false>);
  for_lanes(2 * a.bins + s.count, a.pieces, [&](int64_t first, int64_t n, dim3 grid) {
    a.first = first;
    a.count = n;
    rows<<<grid, dim3(kThreads), 0, stream>>>(a);
  });
  if (const int rc = check_launch("embedding_bwd")) return rc;
  if (a.bins == 0) return 0;
  auto join = accumulate
                  ? (whole ? join_pieces<O, C, true, true> : join_pieces<O, C, false, true>)
                  : (whole ? join_pieces<O, C, true, false> : join_pieces<O, C, false, false>);
  a.pieces = (a.pieces + kWave - 1) / kWave;  // workgroups per row
  a.by_pieces = div_magic(a.pieces);
  const int64_t step = std::max<int64_t>(1, kLanes / kThreads / a.pieces);
  for (a.first = 0; a.first < a.bins; a.first += step) {
    const int64_t n = std::min(step, a.bins - a.first) * a.pieces;
    join<<<dim3(static_cast<unsigned>(n)), dim3(kThreads), 0, stream>>>(a);
  }
  return check_launch("embedding_bwd");
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
  if (count < 0 || width <= 0 || vocab <= 0 || hipo::few_tokens(count, width, vocab)) return 0;
  return hipo::layout(count, width).bytes;
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
  // A workgroup counts its lanes' columns past the last, a batch of places past
  // the end, in 32 bits.
  constexpr int64_t kMost = 0x7fffffff - 4096;
  HIPO_REQUIRE(count <= kMost && width <= kMost && vocab <= (1 << 30),
               "embedding_bwd: count or width over 2^31 - 4097 or vocab over 2^30");
  if (width == 0 || vocab == 0) return 0;
  HIPO_REQUIRE(dweight != nullptr && (count == 0 || (grad != nullptr && tokens != nullptr)),
               "embedding_bwd: null pointer");
  BwdArgs a{};
  a.grad = grad;
  a.dw = dweight;
  a.width = static_cast<int>(width);
  a.scale = scale;
  SortArgs s{};
  s.tokens = tokens;
  s.count = count;
  s.vocab = vocab;
  s.padding_idx = padding_idx;
  if (!accumulate) {
    s.fill = static_cast<uint16_t*>(dweight);
    s.fill_values = vocab * width * (out_size / 2);
  }
  const auto run = [&](auto launch) {
    if (elem_size == 2)
      return out_size == 2 ? launch(uint16_t{}, uint16_t{}) : launch(uint16_t{}, float{});
    return out_size == 2 ? launch(float{}, uint16_t{}) : launch(float{}, float{});
  };
  if (few_tokens(count, width, vocab)) {
    return run([&](auto t, auto o) {
      return launch_few<decltype(t), decltype(o)>(a, s, token_size, accumulate != 0, stream);
    });
  }
  const Layout l = layout(count, width);
  HIPO_REQUIRE(workspace != nullptr && workspace_bytes >= l.bytes,
               "embedding_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, l.bytes);
  HIPO_REQUIRE(aligned16(workspace), "embedding_bwd: workspace must be 16-byte aligned");
  char* ws = static_cast<char*>(workspace);
  s.order = reinterpret_cast<Place*>(ws);
  s.total = reinterpret_cast<int*>(ws + l.total);
  a.order = s.order;
  a.total = s.total;
  a.sums = reinterpret_cast<float*>(ws + l.sums);
  a.bins = l.bins;
  a.bits = l.bits;
  while ((int64_t{1} << s.group_bits) < kSortGroups ||
         (int64_t{kSortRows} << s.group_bits) < vocab) {
    ++s.group_bits;
  }
  return run([&](auto t, auto o) {
    return launch_bwd<decltype(t), decltype(o)>(a, s, token_size, accumulate != 0, stream);
  });
}
