// Softmax cross entropy of the output layer without its logits, and its
// gradients.
//
// With s_j = scale hidden weight_j:  lse = ln sum_j e^(s_j),  loss = lse - s_t;
// d_j = scale ((g + g_lse) e^(s_j - lse) - g [j = t]),  dhidden = d weight,
// dweight = d^T hidden.
//
// Of more than 64 rows all products run through one matrix-product kernel,
// gemm(), of bf16 operands; what becomes of a tile of the result is its epilogue: a
// tile's logits are reduced to one maximum and one sum per row (forward), turned
// into d (backward), or are a tile of a gradient.  Rows that are left out are
// compacted away first, on the device.  The gradient goes through the vocabulary in
// pieces, so that d's piece alone is ever in memory.  The matrix cores bound it:
// 8192 x 4096 x 65536 takes 3.06 ms forward (1.44 PFLOP/s; the library's product
// alone of 8192 x 4096 x 64000: 1.43) and 9.7 backward (1.36).  Up to 64 rows the
// weight's bytes bound everything, and kernels of their own read it as it lies.
//
// fp32 operands are split into three bf16 parts (8 bits of the significand each)
// and multiplied as six products of parts, the smallest first; the three left out
// are below 2^-24 of the largest.  (The fp32 matrix instructions reach a sixteenth
// of the bf16 rate, six products 2.7 times as much.)
//
// d of bf16 operands is rounded to bf16 for its products with them, which the
// matrix cores take of one type: each value is off by half a step (2^-9 of it on
// average), as much again as the gradients' own rounding (relative 2-norms 0.0024
// where gradients rounded from exact d have 0.0017); sums are fp32 throughout.
// Where the caller asks for two parts (and always up to 64 rows) d is held in two
// bf16 parts, some 2^-17 of it, each multiplied: 0.0017 again, at twice the products
// of dhidden and dweight (8192 x 4096 x 128000 16.8 -> 28.9 ms).
#include <algorithm>

#include "hipo_common.h"

namespace hipo {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef u32x2_t u32x2_a2_t __attribute__((aligned(2)));

constexpr int kTile = 256;       // rows of either operand that a workgroup multiplies,
constexpr int kSmallTile = 128;  // or where there are too few such tiles
constexpr int kStep = 64;        // values of K per round
constexpr int kThinRows = 64;    // at most, for the kernels of few rows
constexpr int kSelectRows = 2048;  // at most, for one launch that selects and copies
constexpr int64_t kCus = 256;
constexpr float kLargest = 3.402823466e+38f;

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ---------------------------------------------------------------------------
// Operands: rows that count, and copies in the layout that gemm() reads.
// ---------------------------------------------------------------------------

__device__ __forceinline__ int64_t token_at(const void* tokens, int size, int64_t i) {
  return size == 8 ? static_cast<const int64_t*>(tokens)[i]
                   : static_cast<const int32_t*>(tokens)[i];
}

struct Select {
  const void* tokens;
  int token_size;
  int64_t rows, ignore_index;
  int* kept;      // [rows] the rows that count, in order
  int* count;     // how many
  float* target;  // [rows] set to NaN (forward), or null
  float *loss, *lse;
};

// One workgroup; rows that do not count get their zeros here.
__global__ __launch_bounds__(1024) void select_rows(Select a) {
  __shared__ int waves[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int64_t r0 = 0; r0 < a.rows; r0 += 1024) {
    const int64_t r = r0 + threadIdx.x;
    const bool keep = r < a.rows && token_at(a.tokens, a.token_size, r) != a.ignore_index;
    const uint64_t mask = __ballot(keep);
    if (lane == 0) waves[wave] = __popcll(mask);
    __syncthreads();
    int before = base, sum = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += waves[w];
      sum += waves[w];
    }
    if (keep) {
      const int at = before + __popcll(mask & ((uint64_t{1} << lane) - 1));
      a.kept[at] = static_cast<int>(r);
      if (a.target) a.target[at] = __builtin_nanf("");
    } else if (a.loss && r < a.rows) {
      a.loss[r] = 0.0f;
      a.lse[r] = 0.0f;
    }
    base += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) *a.count = base;
}

// The next bf16 parts of two values, the nearest ones, and what they leave.  All
// but the last are kept finite (a value past the largest bf16 leaves the rest to
// the next part, an infinity or NaN to the last).
__device__ __forceinline__ uint32_t next_parts(float& lo, float& hi, bool last) {
  constexpr float kLargestBf16 = 3.3895313892515355e38f;
  const uint32_t w = last ? pack_bf16x2(lo, hi)
                          : pack_bf16x2(__builtin_amdgcn_fmed3f(lo, -kLargestBf16, kLargestBf16),
                                        __builtin_amdgcn_fmed3f(hi, -kLargestBf16, kLargestBf16));
  lo -= bf16lo(w);
  hi -= bf16hi(w);
  return w;
}

struct Pack {
  const void* src;
  int64_t ld;       // of src
  const int* kept;  // rows of src, or null: all
  const int* count; // how many rows, or null: rows
  int64_t rows;
  int cols;
  uint16_t* dst;
  int64_t dst_ld, plane;  // of dst, in values
  // Where a row's token is ignore_index, it gets zeros in `zero` (or null).
  const void* tokens;
  int token_size;
  int64_t ignore_index;
  void* zero;
};

// 8 values of a row from column k on, zeros from `width` on.
template <typename T>
struct Piece;
template <>
struct Piece<uint16_t> {
  u32x4_t w;
  template <bool Once = false>
  __device__ __forceinline__ void load(const uint16_t* row, int k, int width) {
    if (k + 8 <= width) {
      const u32x4_a2_t* at = reinterpret_cast<const u32x4_a2_t*>(row + k);
      w = Once ? __builtin_nontemporal_load(at) : *at;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = k + 2 * i < width ? row[k + 2 * i] : 0;
        const uint32_t hi = k + 2 * i + 1 < width ? row[k + 2 * i + 1] : 0;
        w[i] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void store(uint16_t* to, int64_t) const {
    *reinterpret_cast<u32x4_t*>(to) = w;
  }
};
template <>
struct Piece<float> {
  f32x4_t v[2];
  template <bool Once = false>
  __device__ __forceinline__ void load(const float* row, int k, int width) {
    if (k + 8 <= width) {
      v[0] = *reinterpret_cast<const f32x4_a4_t*>(row + k);
      v[1] = *reinterpret_cast<const f32x4_a4_t*>(row + k + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = k + i < width ? row[k + i] : 0.0f;
    }
  }
  __device__ __forceinline__ void store(uint16_t* to, int64_t plane) const {
    f32x4_t x[2] = {v[0], v[1]};
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      u32x4_t w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo = x[i >> 1][(2 * i) & 3], hi = x[i >> 1][(2 * i + 1) & 3];
        w[i] = next_parts(lo, hi, q == 2);
        x[i >> 1][(2 * i) & 3] = lo;
        x[i >> 1][(2 * i + 1) & 3] = hi;
      }
      *reinterpret_cast<u32x4_t*>(to + q * plane) = w;
    }
  }
};

// dst[plane][row][0 : dst_ld] = the parts of a row of src, zeros past its end.
template <typename T>
__global__ __launch_bounds__(256) void pack_rows(Pack a) {
  const int64_t rows = a.count ? *a.count : a.rows;
  const int chunks = static_cast<int>(a.dst_ld / 8);
  if (a.zero) {
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
      if (token_at(a.tokens, a.token_size, row) != a.ignore_index) continue;
      for (int c = threadIdx.x; c < a.cols; c += 256) {
        static_cast<T*>(a.zero)[row * a.cols + c] = 0;
      }
    }
  }
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* from = static_cast<const T*>(a.src) + (a.kept ? a.kept[row] : row) * a.ld;
    for (int c = threadIdx.x; c < chunks; c += 256) {
      Piece<T> piece;
      piece.load(from, c * 8, a.cols);
      piece.store(a.dst + row * a.dst_ld + c * 8, a.plane);
    }
  }
}

// select_rows() and pack_rows() at once, for up to kSelectRows rows: each row's
// workgroup counts those before it.  Calls of 8, 512 and 2000 rows take 2.4, 1.5 and
// 1.3 us less, of 4000 rows 1.2 more.
template <typename T>
__global__ __launch_bounds__(256) void select_and_pack_rows(Select s, Pack a) {
  __shared__ int waves[4];
  const int row = blockIdx.x;
  int before = 0;
  for (int r = threadIdx.x; r < row; r += 256) {
    before += token_at(s.tokens, s.token_size, r) != s.ignore_index;
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) before += __shfl_xor(before, o);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = before;
  __syncthreads();
  before = waves[0] + waves[1] + waves[2] + waves[3];
  const bool keep = token_at(s.tokens, s.token_size, row) != s.ignore_index;
  if (threadIdx.x == 0) {
    if (keep) {
      s.kept[before] = row;
      if (s.target) s.target[before] = __builtin_nanf("");
    } else if (s.loss) {
      s.loss[row] = 0.0f;
      s.lse[row] = 0.0f;
    }
    if (row + 1 == s.rows) *s.count = before + keep;
  }
  if (keep) {
    const T* from = static_cast<const T*>(a.src) + row * a.ld;
    for (int k = threadIdx.x * 8; k < a.dst_ld; k += 256 * 8) {
      Piece<T> piece;
      piece.load(from, k, a.cols);
      piece.store(a.dst + before * a.dst_ld + k, a.plane);
    }
  } else if (a.zero) {
    T* to = static_cast<T*>(a.zero) + static_cast<int64_t>(row) * a.cols;
    for (int c = threadIdx.x; c < a.cols; c += 256) to[c] = 0;
  }
}

// ---------------------------------------------------------------------------
// The product of the rows of two matrices
// ---------------------------------------------------------------------------

enum Epilogue { kReduce, kLogitGrad, kAccumulate, kStore };

struct Product {
  // out[j][i] = sum_k a[i][k] b[j][k], where a and b may lie as [k][i] and [k][j].
  // `k` values of K, of which a has a_k rows where it lies as [k][i].  b_count,
  // k_count: read on the device where they are the number of rows that count.
  const uint16_t *a, *b;
  int64_t lda, ldb, a_plane, b_plane;
  int a_rows, b_rows, k, a_k;
  const int *b_count, *k_count;

  // kReduce, kLogitGrad: a is the vocabulary from `first` on, b the rows.
  const void* tokens;
  int token_size;
  const int* kept;
  int64_t first;
  float scale;
  float2* part;  // [tile of the vocabulary][part_ld] maximum and sum
  int64_t part_ld, first_tile;
  float* target;
  const float *grad, *lse, *grad_lse;
  uint16_t* d;  // [rows][d_ld] and its planes
  int64_t d_ld, d_plane, vocab;

  // kAccumulate: sums of the pieces [split][rows][sum_ld], K being split (`to_out`:
  // not split, and the last piece).  kStore: out alone.
  int splits;
  float* sum;
  int64_t sum_ld, sum_plane;
  int load_sum, to_out;
  void* out;
  int64_t out_ld;
};

typedef __attribute__((address_space(3))) const uint16_t* lds_ptr_t;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_t;
typedef int s32x4_t __attribute__((ext_vector_type(4)));

// 16 bytes a lane from byte `from` of the buffer (from its end on: zeros), plus
// the scalar `offset`, to LDS from byte `to` on, lane after lane.  No register is
// written; it is waited for by count, in barrier().  (Of the builtin the compiler
// would wait for every load that might write what an LDS read reads.)  m0 needs
// one wait state before its use.  The compiler keeps nothing in m0 from one
// instruction to another and warns of its name below; but it merges settings of m0
// that it takes to be alike, which this one must end.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(s32x4_t buffer, uint32_t from, int offset,
                                            uint32_t to) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(
                   from),
               "s"(buffer), "s"(offset), "s"(to)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// All but `Loads` loads of this wave and all its LDS reads are done, in every
// wave of the workgroup.
template <int Loads>
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(Loads) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// 4 consecutive values of an output row, `n` of them inside.
__device__ __forceinline__ void store4(uint16_t* p, const f32x4_t& v, int n) {
  if (n >= 4) {
    *reinterpret_cast<u32x2_a2_t*>(p) = u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i < n) p[i] = static_cast<uint16_t>(pack_bf16x2(v[i], 0.0f));
    }
  }
}
__device__ __forceinline__ void store4(float* p, const f32x4_t& v, int n) {
  if (n >= 4) {
    *reinterpret_cast<f32x4_a4_t*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (i < n) p[i] = v[i];
    }
  }
}

// The parts of a and b that are multiplied, the smallest products first: six of
// three parts each, or those of b alone.
__device__ __forceinline__ int a_part(int pass, int passes) {
  return passes == 6 ? (0x001120 >> (4 * pass)) & 3 : 0;
}
__device__ __forceinline__ int b_part(int pass, int passes) {
  return passes == 6 ? (0x010102 >> (4 * pass)) & 3 : passes == 2 ? 1 - pass : 0;
}

// One operand's part of a round: Tile rows by kStep values of K in LDS, moved
// there straight from memory, 16 bytes a lane, 4 instructions a wave.
//
// Of [row][k]: an instruction moves 8 rows of 64 values.  The 16-byte piece c of
// row r lies at place c ^ (r % 8) of its row, so that the 16 rows that a matrix
// instruction's operand is read from lie in different banks.
//
// Of [k][row] (Across): an instruction moves all rows of 2 (Tile 128: 4) values of
// K; the piece c of value k lies at place c ^ (k % 4 * 2), and the operand is read by the
// LDS's transposing loads, 16 lanes of which take 4 values of K of 16 rows.
//
// Two rounds' parts lie one behind the other, from element `first` of the
// workgroup's LDS on.
template <int Tile, bool Across>
struct Operand {
  static constexpr int kWaves = Tile / 32, kPieces = Tile / 8, kValues = 512 / Tile;
  uint32_t from;                // byte of the tile that this lane loads first
  uint32_t at[Across ? 4 : 2];  // element of the LDS that it reads first
  uint32_t to;                  // byte of the LDS that this wave writes first
  int64_t ld, plane;
  const uint16_t* base;
  int valid;   // rows
  int k_rows;  // Across: values of K there are
  int next;    // bytes between instructions

  __device__ __forceinline__ void init(const uint16_t* m, int64_t m_ld, int64_t m_plane, int tile,
                                       int rows, int k, int wave, int lane, int wave_row,
                                       const uint16_t* lds, int first) {
    ld = m_ld;
    plane = m_plane;
    // Across: whole 16-byte pieces, as a load that crosses the buffer's end loses
    // the 4 bytes that do.  (Rows of memory are whole pieces long.)
    valid = min(Tile, (Across ? (rows + 7) / 8 * 8 : rows) - tile * Tile);
    k_rows = k;
    base = m + static_cast<int64_t>(tile) * Tile * (Across ? 1 : ld);
    const uint32_t lds_byte = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr_t)lds));
    to = __builtin_amdgcn_readfirstlane(lds_byte + first * 2 + wave * 1024);
    const int l = lane & 15, g = lane >> 4;
    if constexpr (Across) {
      const int kr = wave * kValues + lane / kPieces;
      from = static_cast<uint32_t>(kr * ld * 2 + ((lane % kPieces) ^ ((kr & 3) << 1)) * 16);
      next = static_cast<int>(kWaves * kValues * ld * 2);
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        at[f] = first + (g * 8 + (l >> 2)) * Tile + wave_row +
                ((2 * f + ((l & 3) >> 1)) ^ ((l >> 2) << 1)) * 8 + (l & 1) * 4;
        // (Else `first` joins the reads' offsets, which hold 16 bits.)
        asm volatile("" : "+v"(at[f]));
      }
    } else {
      const int row = wave * 8 + (lane >> 3);
      from = static_cast<uint32_t>(row * ld * 2 + ((lane & 7) ^ (lane >> 3)) * 16);
      next = static_cast<int>(kWaves * 8 * ld * 2);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        at[h] = first + (wave_row + l) * kStep + (((h * 4 + g) ^ (l & 7)) * 8);
        asm volatile("" : "+v"(at[h]));
      }
    }
  }

  struct Round {
    s32x4_t buffer;
    int offset;
    uint32_t from;
  };

  // The round of K from k0 on; from k on there are zeros.
  __device__ __forceinline__ Round round(int part, int k0, int k, int lane) const {
    const uint16_t* here = base + part * plane;
    int bytes, offset;
    uint32_t first = from;
    if constexpr (Across) {
      // Rows of K past the last are past the buffer's end, which reads as zero.
      const int left = min(kStep, k_rows - k0);
      bytes = max(0, static_cast<int>(((left - 1) * ld + valid) * 2));
      bytes = left > 0 ? bytes : 0;
      offset = 0;
      here += min(k0, k_rows) * ld;
    } else {
      bytes = static_cast<int>(((valid - 1) * ld + k) * 2);
      offset = k0 * 2;
      first |= k0 + ((lane & 7) ^ (lane >> 3)) * 8 < k ? 0u : 0x80000000u;
    }
    const uint64_t address = reinterpret_cast<uint64_t>(here);
    const s32x4_t r = {__builtin_amdgcn_readfirstlane(static_cast<int>(address)),
                       __builtin_amdgcn_readfirstlane(static_cast<int>(address >> 32) & 0xffff),
                       __builtin_amdgcn_readfirstlane(bytes), 0x00027000};
    return Round{r, __builtin_amdgcn_readfirstlane(offset), first};
  }

  // A quarter of it.
  __device__ __forceinline__ void load(int buffer, int q, const Round& r) const {
    load_to_lds(r.buffer, r.from + q * next, r.offset,
                to + buffer * Tile * kStep * 2 + q * kWaves * 1024);
  }

  // Rows 16 f to 16 f + 15 of the wave's, 32 values of K of half `h`: row l, values
  // 8 g to 8 g + 7 for lane 16 g + l.
  __device__ __forceinline__ bf16x8_t fetch(const uint16_t* lds, int buffer, int h, int f) const {
    if constexpr (Across) {
      const uint16_t* p = lds + at[f & 3] + buffer * Tile * kStep + (f >> 2) * 64 + h * 32 * Tile;
      const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)p);
      const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(p + 4 * Tile));
      const auto both = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(bf16x8_t, both);
    } else {
      return *reinterpret_cast<const bf16x8_t*>(lds + at[h] + buffer * Tile * kStep +
                                                f * 16 * kStep);
    }
  }
};

// Tile / 32 waves, 2 by Tile / 64, of Tile / 2 by 64 values each.
//
// What it took (8192 x 4096 x 65536, eighth of the rows left out, forward): loads to
// LDS a round ahead with two barriers a round 1.14 PFLOP/s; the operands of half a
// round in registers ahead and one barrier 1.29; loads and LDS reads spread among
// the matrix instructions 1.45.  LDS reads of the 256 tile take 1536 of a round's
// 2048 cycles; 131 KB of LDS and 240 registers leave one workgroup a CU.  At 1.8 GHz,
// where the card's power holds it, the matrix cores were busy 65 % of the cycles
// before the last step.  No gain: s_setprio around the products, bands of 8 tiles
// instead of 4 for an XCD, rows of copies and of d padded off powers of two.
//
// Parts: of d, which kLogitGrad writes and the gradients' products read as b.
template <typename T, int Tile, Epilogue E, int Parts = sizeof(T) == 2 ? 1 : 3>
__global__ __launch_bounds__(Tile * 2, 2) void gemm(Product p) {
  constexpr int kWavesB = Tile / 64, kFragments = Tile / 32;
  constexpr bool kOfD = E == kAccumulate || E == kStore;
  constexpr int kPasses = sizeof(T) == 4 ? 6 : kOfD ? Parts : 1;
  constexpr bool kAcrossA = kOfD, kAcrossB = E == kStore;
  __shared__ __attribute__((aligned(1024))) uint16_t lds[4 * Tile * kStep];

  const int rows_b = p.b_count ? *p.b_count : p.b_rows;
  const int k = p.k_count ? *p.k_count : p.k;
  // Tiles in an order that keeps an XCD's workgroups on 4 tiles of a by 8 of b.
  const int tiles_a = (p.a_rows + Tile - 1) / Tile;
  const int tiles_b = (rows_b + Tile - 1) / Tile;
  const uint32_t tiles = static_cast<uint32_t>(tiles_a) * tiles_b;
  const uint32_t all = tiles * p.splits;  // an XCD's share of them is of one split or two
  if (blockIdx.x >= all) return;
  const uint32_t place = xcd_order(blockIdx.x, all);
  const uint32_t split = place / tiles, id = place % tiles;
  const int band = id / (4 * tiles_b), in_band = id % (4 * tiles_b);
  const int band_rows = min(4, tiles_a - band * 4);
  const int tile_a = band * 4 + in_band % band_rows, tile_b = in_band / band_rows;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int valid_b = min(Tile, rows_b - tile_b * Tile);
  const int wave_a = wave / kWavesB * (Tile / 2), wave_b = wave % kWavesB * 64;
  Operand<Tile, kAcrossA> oa;
  Operand<Tile, kAcrossB> ob;
  oa.init(p.a, p.lda, p.a_plane, tile_a, p.a_rows, p.k_count ? k : p.a_k, wave, lane, wave_a,
          lds, 0);
  ob.init(p.b, p.ldb, p.b_plane, tile_b, rows_b, k, wave, lane, wave_b, lds,
          2 * Tile * kStep);

  f32x4_t acc[kFragments][4];  // of 16 by 16 values
#pragma unroll
  for (int f = 0; f < kFragments; ++f) {
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[f][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // A round is two halves of 32 values of K; a half's operands are read from LDS
  // into one set of registers while the other set is multiplied.
  bf16x8_t fa[2][kFragments], fb[2][4];

  // Rounds of K, in pairs.  Rounds past the last (the second of an odd pair, and
  // the two loaded behind the end) load zeros.
  int begin = 0, end = (k + kStep - 1) / kStep;
  if (E == kAccumulate) {
    // (Divided by lanes: back to scalars, which the loads need.)
    const int64_t whole = end;
    begin = __builtin_amdgcn_readfirstlane(static_cast<int>(whole * split / p.splits));
    end = __builtin_amdgcn_readfirstlane(static_cast<int>(whole * (split + 1) / p.splits));
  }
  const int rounds = (end - begin) * kPasses;
  int pass = 0, at = begin;
  typename Operand<Tile, kAcrossA>::Round ra;
  typename Operand<Tile, kAcrossB>::Round rb;
  auto prepare = [&]() __attribute__((always_inline)) {
    const int k0 = pass < kPasses ? at * kStep : max(k, p.a_k);
    const int now = min(pass, kPasses - 1);
    ra = oa.round(a_part(now, kPasses), k0, k, lane);
    rb = ob.round(b_part(now, kPasses), k0, k, lane);
    const bool wrap = ++at >= end;
    at = wrap ? begin : at;
    pass += wrap ? 1 : 0;
  };
  // The products of half `half`, in groups; with each a part of what the other
  // half needs is read from LDS and a load of the round after next begins, so that
  // neither waits in a row for the units that take them.
  auto multiply = [&](int half, int buffer, bool load) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < kFragments; ++f) {
      constexpr int kLoads = 8 / kFragments, kReads = kFragments == 8 ? 2 : 3;
      if (load) {
#pragma unroll
        for (int q = f * kLoads; q < (f + 1) * kLoads; ++q) {
          if (q < 4) {
            oa.load(buffer, q, ra);
          } else {
            ob.load(buffer, q - 4, rb);
          }
        }
      }
      const int from = load ? buffer ^ 1 : buffer;
#pragma unroll
      for (int m = kReads * f; m < min(kReads * (f + 1), kFragments + 4); ++m) {
        if (m < 4) {
          fb[half ^ 1][m] = ob.fetch(lds, from, half ^ 1, m);
        } else {
          fa[half ^ 1][m - 4] = oa.fetch(lds, from, half ^ 1, m - 4);
        }
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        acc[f][n] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[half][f], fb[half][n], acc[f][n], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // One barrier a round: behind it the round's buffer is read and free for the
  // round after next, and the next round's loads have arrived.
  auto round = [&](int buffer) __attribute__((always_inline)) {
    prepare();
    multiply(0, buffer, false);
    barrier<0>();
    multiply(1, buffer, true);
  };
  // (5 wait states from a vector instruction's scalar result to a load.)
  auto load_all = [&](int buffer) __attribute__((always_inline)) {
    prepare();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 4");
#pragma unroll
    for (int q = 0; q < 4; ++q) oa.load(buffer, q, ra);
#pragma unroll
    for (int q = 0; q < 4; ++q) ob.load(buffer, q, rb);
  };
  load_all(0);
  load_all(1);
  barrier<8>();
#pragma unroll
  for (int n = 0; n < 4; ++n) fb[0][n] = ob.fetch(lds, 0, 0, n);
#pragma unroll
  for (int f = 0; f < kFragments; ++f) fa[0][f] = oa.fetch(lds, 0, 0, f);
  for (int t = 0; t < rounds; t += 2) {
    round(0);
    round(1);
  }
  barrier<0>();

  // acc[f][n][r] is out[j][i] with these.
  const int i0 = tile_a * Tile + wave_a + (lane >> 4) * 4;  // + 16 f + r
  const int j0 = tile_b * Tile + wave_b + (lane & 15);      // + 16 n

  if (E == kReduce) {
    // A row's values are 4 kFragments of each of 4 lanes in each of 2 waves; a maximum and
    // a sum of e^(s - maximum) of each, in units of the logits without `scale`
    // (which is positive) up to the end.
    float* both = reinterpret_cast<float*>(lds);  // [wave_a][2][Tile]
    const float to_log2 = p.scale * kLog2eHi;
    if (tile_a + 1 == tiles_a) {
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (i0 + f * 16 + r >= p.a_rows) acc[f][n][r] = -INFINITY;
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = j0 + n * 16;
      int64_t tok = -1;
      if (j < rows_b) tok = token_at(p.tokens, p.token_size, p.kept[j]) - p.first - i0;
      if (tok >= 0 && tok < kFragments * 16 - 12 && i0 + tok < p.a_rows) {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (tok == f * 16 + r) p.target[j] = acc[f][n][r] * p.scale;
          }
        }
      }
      float top = -kLargest;
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[f][n][r]);
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      top = fminf(top, kLargest);
      float sum = 0.0f;
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sum += __builtin_amdgcn_exp2f((acc[f][n][r] - top) * to_log2);
        }
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane < 16) {
        both[(wave / kWavesB * 2 + 0) * Tile + wave_b + n * 16 + lane] = top * p.scale;
        both[(wave / kWavesB * 2 + 1) * Tile + wave_b + n * 16 + lane] = sum;
      }
    }
    __syncthreads();
    if (threadIdx.x < Tile && static_cast<int>(threadIdx.x) < valid_b) {
      const int j = threadIdx.x;
      const float t0 = both[j], s0 = both[Tile + j];
      const float t1 = both[2 * Tile + j], s1 = both[3 * Tile + j];
      const float top = fmaxf(t0, t1);
      const float sum = s0 * exp_f32(exp_domain(t0 - top)) + s1 * exp_f32(exp_domain(t1 - top));
      p.part[(p.first_tile + tile_a) * p.part_ld + tile_b * Tile + j] = make_float2(top, sum);
    }
  }

  if (E == kLogitGrad) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = j0 + n * 16;
      float g = 0.0f, both = 0.0f, lse = 0.0f;  // of rows past the last, whose products are 0
      int64_t tok = -1;
      if (j < rows_b) {
        const int row = p.kept[j];
        tok = token_at(p.tokens, p.token_size, row);
        g = p.grad[row];
        if (tok < 0 || tok >= p.vocab) g = __builtin_nanf("");
        both = p.grad_lse ? g + p.grad_lse[row] : g;
        lse = p.lse[row];
        tok -= p.first + i0;
      }
      both *= p.scale;
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float ln_p = __builtin_fmaf(acc[f][n][r], p.scale, -lse);
          acc[f][n][r] = both * __builtin_amdgcn_exp2f(ln_p * kLog2eHi);
        }
      }
      if (tok >= 0 && tok < kFragments * 16 - 12) {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (tok == f * 16 + r) acc[f][n][r] -= g * p.scale;
          }
        }
      }
    }
    if (tile_a + 1 == tiles_a) {
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (i0 + f * 16 + r >= p.a_rows) acc[f][n][r] = 0.0f;
          }
        }
      }
    }
  }

  if constexpr (E == kLogitGrad || (E == kStore && sizeof(T) == 2)) {
    // bf16 through LDS, so that 32 lanes (Tile 128: 16) store consecutive bytes of
    // a row (straight from the registers a store is 32 bytes of each of 16 rows: the
    // gradients of 256 x 4096 x 128000 took 0.72 ms for dweight's 1 GB).  The
    // 16-byte piece c of row j lies at place c ^ (j % pieces).
    constexpr int kPieces = Tile / 8, kValues = 512 / Tile;
#pragma unroll
    for (int q = 0; q < (E == kLogitGrad ? Parts : 1); ++q) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int j = wave_b + n * 16 + (lane & 15);
#pragma unroll
        for (int f = 0; f < kFragments; ++f) {
          const int i = wave_a + f * 16 + (lane >> 4) * 4;
          u32x2_t v;
          if (E == kStore || Parts == 1) {
            v = u32x2_t{pack_bf16x2(acc[f][n][0], acc[f][n][1]),
                        pack_bf16x2(acc[f][n][2], acc[f][n][3])};
          } else {
            float x[4] = {acc[f][n][0], acc[f][n][1], acc[f][n][2], acc[f][n][3]};
            constexpr int kLast = Parts - 1;
            v = u32x2_t{next_parts(x[0], x[1], q == kLast), next_parts(x[2], x[3], q == kLast)};
            acc[f][n] = f32x4_t{x[0], x[1], x[2], x[3]};
            asm volatile("" : "+v"(acc[f][n]));  // what is left takes its place: no spills
          }
          *reinterpret_cast<u32x2_t*>(lds + j * Tile + (((i >> 3) ^ (j % kPieces)) << 3) +
                                      (i & 7)) = v;
        }
      }
      __syncthreads();
      const int piece = lane % kPieces;
      const int i = tile_a * Tile + piece * 8;
#pragma unroll 4
      for (int r = 0; r < Tile; r += kFragments * kValues) {
        const int j = r + wave * kValues + lane / kPieces;
        const u32x4_t v =
            *reinterpret_cast<const u32x4_t*>(lds + j * Tile + ((piece ^ (j % kPieces)) << 3));
        if (E == kLogitGrad) {
          *reinterpret_cast<u32x4_t*>(p.d + q * p.d_plane +
                                      (tile_b * static_cast<int64_t>(Tile) + j) * p.d_ld + i) = v;
        } else if (j < valid_b) {
          uint16_t* out = static_cast<uint16_t*>(p.out) +
                          (tile_b * static_cast<int64_t>(Tile) + j) * p.out_ld + i;
          if (i + 8 <= p.a_rows) {
            // (Of no use in the caches: 256 x 4096 x 128000 1034 -> 971 us, with the
            // rows of few-row calls 732 -> 690.)
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4_a2_t*>(out));
          } else {
#pragma unroll
            for (int m = 0; m < 7; ++m) {
              if (i + m < p.a_rows) out[m] = static_cast<uint16_t>(v[m >> 1] >> (m & 1) * 16);
            }
          }
        }
      }
      __syncthreads();
    }
  } else if constexpr (E == kAccumulate || E == kStore) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int j = j0 + n * 16;
      asm volatile("" ::: "memory");  // no loads of later rows ahead of this one's
      if (j >= rows_b) continue;
      T* out = static_cast<T*>(p.out) +
               static_cast<int64_t>(E == kStore ? j : (p.to_out ? p.kept[j] : 0)) * p.out_ld;
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
        const int i = i0 + f * 16;
        if (i >= p.a_rows) continue;
        f32x4_t v = acc[f][n];
        if (E == kAccumulate) {
          f32x4_t* sum = reinterpret_cast<f32x4_t*>(p.sum + split * p.sum_plane +
                                                     j * p.sum_ld + i);
          if (p.load_sum) v += *sum;
          if (!p.to_out) {
            *sum = v;
            continue;
          }
        }
        store4(out + i, v, p.a_rows - i);
      }
    }
  }
}

struct JoinLoss {
  const float2* part;
  int64_t part_ld;
  int tiles;
  const int *kept, *count;
  const float* target;
  float *loss, *lse;
};

// One tile's maximum and sum joined to the ones so far, and the loss of a row:
// with the logit's distance from the maximum, which is exact where they are near.
__device__ __forceinline__ void join_one(float& top, float& sum, float2 v) {
  const float m = fmaxf(top, v.x);
  sum = sum * exp_f32(exp_domain(top - m)) + v.y * exp_f32(exp_domain(v.x - m));
  top = m;
}

__device__ __forceinline__ void put_loss(float top, float sum, float target, float* loss,
                                         float* lse) {
  const float log_sum = logf(sum);
  *lse = top + log_sum;
  *loss = log_sum - (target - top);
}

// 16 rows by 16 parts of the vocabulary's tiles per workgroup.
__global__ __launch_bounds__(256) void join_loss(JoinLoss a) {
  __shared__ float2 parts[16][16];
  const int count = *a.count;
  const int row = threadIdx.x & 15, part = threadIdx.x >> 4;
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * 16; first < count;
       first += static_cast<int64_t>(gridDim.x) * 16) {
    const int64_t j = first + row;
    float top = -kLargest, sum = 0.0f;
    if (j < count) {
#pragma unroll 8
      for (int t = part; t < a.tiles; t += 16) join_one(top, sum, a.part[t * a.part_ld + j]);
    }
    parts[part][row] = make_float2(top, sum);
    __syncthreads();
    if (part == 0 && j < count) {
      for (int q = 1; q < 16; ++q) join_one(top, sum, parts[q][row]);
      put_loss(top, sum, a.target[j], a.loss + a.kept[j], a.lse + a.kept[j]);
    }
    __syncthreads();
  }
}

// The splits' sums added in order: rows of dhidden.
template <typename T>
__global__ __launch_bounds__(256) void join_hidden(const float* sum, int64_t sum_ld,
                                                   int64_t sum_plane, int splits, bool two_parts,
                                                   const int* kept, const int* count, T* out,
                                                   int width) {
  const int chunks = (width + 3) / 4;
  const int64_t n = static_cast<int64_t>(*count) * chunks;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < n;
       t += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t j = t / chunks;
    const int i = static_cast<int>(t % chunks) * 4;
    const float* from = sum + j * sum_ld + i;
    f32x4_t v = *reinterpret_cast<const f32x4_t*>(from);
#pragma unroll 8
    for (int q = 1; q < splits; ++q) v += *reinterpret_cast<const f32x4_t*>(from + q * sum_plane);
    if (two_parts) {
      from += kThinRows * sum_ld;
#pragma unroll 8
      for (int q = 0; q < splits; ++q) v += *reinterpret_cast<const f32x4_t*>(from + q * sum_plane);
    }
    store4(out + kept[j] * static_cast<int64_t>(width) + i, v, width - i);
  }
}

// ---------------------------------------------------------------------------
// Few rows: the vocabulary is read once, as it lies
// ---------------------------------------------------------------------------

struct Thin {
  const void *hidden, *weight, *tokens;
  int token_size, rows, width;
  int64_t vocab, hidden_ld, weight_ld;
  float scale;
  float2* part;  // [rows][tiles] maximum and sum
  float* target;
  int64_t tiles;

  // Of the gradient: the rows that count, and d of the vocabulary from `first` on.
  const int *kept, *count;
  const float *grad, *lse, *grad_lse;
  uint16_t* d;
  int64_t d_ld, d_plane, first, whole_vocab;
};

constexpr int kThinTile = 64;   // of the vocabulary
constexpr int kThinStages = 4;  // loads in flight, in rounds of kStep values of K

// bf16 parts of d.  Two of bf16 operands, which cost few rows nothing (memory
// bounds them): with one the gradients of a single row are off by up to twice
// what their own rounding to bf16 is, where one token's d outweighs the others'.
template <typename T>
constexpr int kThinParts = sizeof(T) == 2 ? 2 : 3;
template <typename T>
constexpr int kThinPasses = sizeof(T) == 2 ? 2 : 6;
// The parts of an operand and of d that are multiplied, the smallest products first.
template <typename T>
__device__ __forceinline__ int thin_a_part(int pass) {
  return sizeof(T) == 2 ? 0 : a_part(pass, 6);
}
template <typename T>
__device__ __forceinline__ int thin_d_part(int pass) {
  return sizeof(T) == 2 ? 1 - pass : b_part(pass, 6);
}

// The logits of up to 16 N rows against 64 of the vocabulary per workgroup, 16 a
// wave, reduced or (Grad) turned into d as gemm()'s.  Both operands go through
// registers, kThinStages rounds ahead, to LDS (places as in Operand): the weight is
// read once, at any alignment, fp32 split on the way.  Memory bounds it (1 x 4096 x
// 128000 bf16: 188 us, 5.6 TB/s; fp32 452 us, 4.6): the loads in flight (32 KB a
// workgroup of bf16) and the number of workgroups are what counts.  Where there are
// few, K is split among `Groups` groups of four waves, whose sums are added
// through LDS.  Once: the weight takes no place in the caches.
template <typename T, int N, bool Grad, int Groups, bool Once = false>
__global__ __launch_bounds__(256 * Groups) void thin_logits(Thin a) {
  constexpr int kPlanes = sizeof(T) == 2 ? 1 : 3, kPasses = kPlanes == 1 ? 1 : 6;
  constexpr int kPlaneW = kThinTile * kStep, kPlaneH = 16 * N * kStep;
  constexpr int kPiecesH = (N + 1) / 2;
  __shared__ __attribute__((aligned(16))) uint16_t weights[Groups][2][kPlanes * kPlaneW];
  __shared__ __attribute__((aligned(16))) uint16_t hiddens[Groups][2][kPlanes * kPlaneH];
  __shared__ float2 parts[4][16 * N];
  const int group = threadIdx.x >> 8, thread = threadIdx.x & 255;
  uint16_t(&weight)[2][kPlanes * kPlaneW] = weights[group];
  uint16_t(&hidden)[2][kPlanes * kPlaneH] = hiddens[group];
  const int lane = thread & 63, wave = thread >> 6;
  const int l = lane & 15, g = lane >> 4;
  const int row = thread >> 3, chunk = thread & 7;
  const int place = row * kStep + ((chunk ^ (row & 7)) * 8);  // and 32 rows on
  const float to_log2 = a.scale * kLog2eHi;
  const bool with_h = N > 1 || thread < 128;
  const int rows = Grad ? *a.count : a.rows;
  if (rows == 0) return;
  // This group's columns: from `begin` to `end`, `length` at most.
  const int length = ((a.width + kStep - 1) / kStep + Groups - 1) / Groups * kStep;
  const int begin = group * length, end = min(a.width, begin + length);
  const T* from_h[kPiecesH];
#pragma unroll
  for (int q = 0; q < kPiecesH; ++q) {
    const int64_t j = min(row + 32 * q, rows - 1);
    from_h[q] = static_cast<const T*>(a.hidden) + (Grad ? a.kept[j] : j) * a.hidden_ld;
  }
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t first = tile * kThinTile;
    const T* from_w[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      from_w[q] = static_cast<const T*>(a.weight) +
                  min(first + row + 32 * q, a.vocab - 1) * a.weight_ld;
    }
    Piece<T> w[kThinStages][2], h[kThinStages][kPiecesH];
    auto load = [&](int stage, int k0) __attribute__((always_inline)) {
      const int k = begin + k0 + chunk * 8;
#pragma unroll
      for (int q = 0; q < 2; ++q) w[stage][q].template load<Once>(from_w[q], k, end);
      if (with_h) {
#pragma unroll
        for (int q = 0; q < kPiecesH; ++q) h[stage][q].load(from_h[q], k, end);
      }
    };
    // Two sums, of the halves of the rounds: shorter ones round less.
    f32x4_t acc[N], other[N];
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = other[n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < kThinStages; ++s) load(s, s * kStep);
    for (int k0 = 0; k0 < length; k0 += kThinStages * kStep) {
#pragma unroll
      for (int s = 0; s < kThinStages; ++s) {
        if (k0 + s * kStep >= length) break;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          w[s][q].store(weight[s & 1] + place + q * 32 * kStep, kPlaneW);
        }
        if (with_h) {
#pragma unroll
          for (int q = 0; q < kPiecesH; ++q) {
            h[s][q].store(hidden[s & 1] + place + q * 32 * kStep, kPlaneH);
          }
        }
        load(s, k0 + (s + kThinStages) * kStep);
        // One barrier a round: a buffer is written again behind the next one's.
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int at = l * kStep + (((half * 4 + g) ^ (l & 7)) * 8);
          bf16x8_t fw[kPlanes], fh[kPlanes][N];
#pragma unroll
          for (int q = 0; q < kPlanes; ++q) {
            fw[q] = *reinterpret_cast<const bf16x8_t*>(weight[s & 1] + q * kPlaneW +
                                                       wave * 16 * kStep + at);
#pragma unroll
            for (int n = 0; n < N; ++n) {
              fh[q][n] = *reinterpret_cast<const bf16x8_t*>(hidden[s & 1] + q * kPlaneH +
                                                            n * 16 * kStep + at);
            }
          }
#pragma unroll
          for (int pass = 0; pass < kPasses; ++pass) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
              f32x4_t& sum = half == 0 ? acc[n] : other[n];
              sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  fw[a_part(pass, kPasses)], fh[b_part(pass, kPasses)][n], sum, 0, 0, 0);
            }
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] += other[n];
    if constexpr (Groups > 1) {
      __syncthreads();
      // In LDS that the group itself has read.
      f32x4_t* sums = reinterpret_cast<f32x4_t*>(weights[group]);
      if (group > 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) sums[n * 256 + thread] = acc[n];
      }
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int q = 1; q < Groups; ++q) {
          const f32x4_t* from = reinterpret_cast<const f32x4_t*>(weights[q]);
#pragma unroll
          for (int n = 0; n < N; ++n) acc[n] += from[n * 256 + thread];
        }
      }
    }
    const int64_t i0 = first + wave * 16 + g * 4;
    if constexpr (Grad) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (group > 0) break;
        const int j = n * 16 + l;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (j < rows) {
          const int64_t at = a.kept[j], tok = token_at(a.tokens, a.token_size, at);
          const float grad = tok >= 0 && tok < a.whole_vocab ? a.grad[at] : __builtin_nanf("");
          const float both = (a.grad_lse ? grad + a.grad_lse[at] : grad) * a.scale;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float ln_p = __builtin_fmaf(acc[n][r], a.scale, -a.lse[at]);
            v[r] = both * __builtin_amdgcn_exp2f(ln_p * kLog2eHi);
            if (i0 + r == tok - a.first) v[r] -= grad * a.scale;
            if (i0 + r >= a.vocab) v[r] = 0.0f;
          }
        }
#pragma unroll
        for (int q = 0; q < kThinParts<T>; ++q) {
          const bool last = q + 1 == kThinParts<T>;
          const uint32_t lo = next_parts(v[0], v[1], last), hi = next_parts(v[2], v[3], last);
          *reinterpret_cast<u32x2_t*>(a.d + q * a.d_plane + j * a.d_ld + i0) = u32x2_t{lo, hi};
        }
      }
      __syncthreads();
      continue;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (group > 0) break;
      const int j = n * 16 + l;
      const int64_t tok = j < a.rows ? token_at(a.tokens, a.token_size, j) : -1;
      float top = -kLargest;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (i0 + r >= a.vocab) acc[n][r] = -INFINITY;
        if (i0 + r == tok && tok < a.vocab) a.target[j] = acc[n][r] * a.scale;
        top = fmaxf(top, acc[n][r]);
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      top = fminf(top, kLargest);
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += __builtin_amdgcn_exp2f((acc[n][r] - top) * to_log2);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (g == 0) parts[wave][j] = make_float2(top * a.scale, sum);
    }
    __syncthreads();
    const int j = threadIdx.x;
    if (j < a.rows) {
      float top = parts[0][j].x, sum = parts[0][j].y;
#pragma unroll
      for (int q = 1; q < 4; ++q) join_one(top, sum, parts[q][j]);
      a.part[j * a.tiles + tile] = make_float2(top, sum);
    }
    __syncthreads();
  }
}

struct ThinWeight {
  const uint16_t *hidden, *d;  // [row][hidden_ld], [row][d_ld] and their planes
  int64_t hidden_ld, hidden_plane, d_ld, d_plane;
  const int* count;
  int width;
  int64_t vocab;
  void* out;
  int64_t out_ld;
  int chunks;  // of 64 columns, per workgroup
};

// dweight of up to 64 rows: 64 of the vocabulary per workgroup, 16 a wave, whose
// d stays in registers while the columns pass, 64 at a time.  The products'
// operands are [row][...], read across as in Operand.  What is written bounds it,
// so several workgroups a CU write at once, whole 128-byte pieces of rows (1 x 4096
// x 128000: 264 us for 1.05 GB, where gemm()'s tiles of one or two rounds took 360).
template <typename T>
__global__ __launch_bounds__(256) void thin_weight(ThinWeight a) {
  constexpr int kPlanes = sizeof(T) == 2 ? 1 : 3, kParts = kThinParts<T>;
  constexpr int kPlane = 64 * 64;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][kParts * kPlane];
  __shared__ __attribute__((aligned(16))) uint16_t stage[4][sizeof(T) == 2 ? 16 * 64 : 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 15, g = lane >> 4;
  const int row = threadIdx.x >> 3, chunk = threadIdx.x & 7;
  const int place = row * 64 + ((chunk ^ ((row & 3) << 1)) * 8);  // and 32 rows on
  const int count = *a.count;
  const int64_t v0 = static_cast<int64_t>(blockIdx.x) * 64;
  const int begin = blockIdx.y * a.chunks * 64;
  const int end = min(begin + a.chunks * 64, (a.width + 63) / 64 * 64);

  u32x4_t piece[kParts][2];
  // 64 columns of the rows that count, zeros for the others, of some planes.
  auto load = [&](const uint16_t* from, int64_t ld, int64_t plane, int planes)
                  __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      if (p >= planes) continue;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = row + 32 * q;
        piece[p][q] = u32x4_t{0u, 0u, 0u, 0u};
        if (r < count) {
          piece[p][q] = *reinterpret_cast<const u32x4_t*>(from + p * plane + r * ld + chunk * 8);
        }
      }
    }
  };
  auto store = [&](int buffer, int planes) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      if (p >= planes) continue;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        *reinterpret_cast<u32x4_t*>(lds[buffer] + p * kPlane + place + q * 32 * 64) = piece[p][q];
      }
    }
  };
  // Columns 16 f to 16 f + 15, rows 32 h to 32 h + 31: column l, rows 8 g on.
  auto fetch = [&](int buffer, int p, int h, int f) __attribute__((always_inline)) {
    const uint16_t* from = lds[buffer] + p * kPlane + (h * 32 + g * 8 + (l >> 2)) * 64 +
                           ((2 * f + ((l & 3) >> 1)) ^ ((l >> 2) << 1)) * 8 + (l & 1) * 4;
    const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)from);
    const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(from + 4 * 64));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  load(a.d + v0, a.d_ld, a.d_plane, kParts);
  store(0, kParts);
  load(a.hidden + begin, a.hidden_ld, a.hidden_plane, kPlanes);
  __syncthreads();
  bf16x8_t fd[2][kParts];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) fd[h][p] = fetch(0, p, h, wave);
  }
  int buffer = 1;
  for (int c0 = begin; c0 < end; c0 += 64, buffer ^= 1) {
    store(buffer, kPlanes);
    load(a.hidden + min(c0 + 64, end - 64), a.hidden_ld, a.hidden_plane, kPlanes);
    // One barrier a round: a buffer is written again behind the next one's.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int64_t v = v0 + wave * 16;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h * 32 >= count) continue;
        bf16x8_t fh[kPlanes];
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) fh[p] = fetch(buffer, p, h, f);
#pragma unroll
        for (int pass = 0; pass < kThinPasses<T>; ++pass) {
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              fh[thin_a_part<T>(pass)], fd[h][thin_d_part<T>(pass)], acc, 0, 0, 0);
        }
      }
      // acc[r] is row v + l, column c0 + 16 f + 4 g + r.
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x2_t*>(stage[wave] + l * 64 + (((2 * f + (g >> 1)) ^ (l & 7)) * 8) +
                                    (g & 1) * 4) =
            u32x2_t{pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
      } else {
        const int i = c0 + 16 * f + 4 * g;
        if (v + l < a.vocab && i < a.width) {
          store4(static_cast<float*>(a.out) + (v + l) * a.out_ld + i, acc, a.width - i);
        }
      }
    }
    if constexpr (sizeof(T) == 2) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // of this wave's own lanes
      const int i = c0 + (lane & 7) * 8;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int j = q * 8 + (lane >> 3);
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(
            stage[wave] + j * 64 + (((lane & 7) ^ (j & 7)) * 8));
        if (v + j >= a.vocab) continue;
        uint16_t* out = static_cast<uint16_t*>(a.out) + (v + j) * a.out_ld + i;
        if (i + 8 <= a.width) {
          __builtin_nontemporal_store(w, reinterpret_cast<u32x4_a2_t*>(out));
        } else {
#pragma unroll
          for (int m = 0; m < 7; ++m) {
            if (i + m < a.width) out[m] = static_cast<uint16_t>(w[m >> 1] >> (m & 1) * 16);
          }
        }
      }
    }
  }
}

struct ThinHidden {
  const void* weight;  // [vocab][weight_ld], as it lies
  int64_t weight_ld, vocab;
  int width;
  const uint16_t* d;  // [row][d_ld] and its planes, zeros past the rows and the vocabulary
  int64_t d_ld, d_plane;
  const int* count;
  float* sum;  // [split][kThinRows][sum_ld]
  int64_t sum_ld;
  int load_sum;
};

// dhidden of up to 16 N rows: 64 columns of a part of the vocabulary per
// workgroup, 16 a wave, the parts joined by join_hidden().  The weight goes
// through registers to LDS (as in thin_logits(), read across as in Operand), two
// rounds of 64 of the vocabulary ahead; its second reading bounds the kernel.  (Of
// aligned bf16 gemm() is quicker, d's parts as 128 rows: 64 x 4096 x 128000 205 us
// against 318.)
template <typename T, int N>
__global__ __launch_bounds__(256) void thin_hidden(ThinHidden a) {
  constexpr int kPlanes = sizeof(T) == 2 ? 1 : 3, kParts = kThinParts<T>;
  constexpr int kPlaneW = 64 * 64, kPlaneD = 16 * N * 64, kPiecesD = (N + 1) / 2;
  __shared__ __attribute__((aligned(16))) uint16_t weight[2][kPlanes * kPlaneW];
  __shared__ __attribute__((aligned(16))) uint16_t ds[2][kParts * kPlaneD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane & 15, g = lane >> 4;
  const int row = threadIdx.x >> 3, chunk = threadIdx.x & 7;
  const int place_w = row * 64 + ((chunk ^ ((row & 3) << 1)) * 8);  // and 32 rows on
  const int place_d = row * 64 + ((chunk ^ (row & 7)) * 8);
  const bool with_d = N > 1 || threadIdx.x < 128;
  const int count = *a.count;
  if (count == 0) return;
  const int c0 = blockIdx.x * 64;
  const int64_t rounds = (a.vocab + 63) / 64;
  const int64_t begin = rounds * blockIdx.y / gridDim.y;
  const int64_t end = rounds * (blockIdx.y + 1) / gridDim.y;

  Piece<T> w[2][2];
  u32x4_t d[2][kParts][kPiecesD];
  auto load = [&](int stage, int64_t t) __attribute__((always_inline)) {
    const int64_t v0 = min(t, end - 1) * 64;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      // (Past the vocabulary, and past a row's end, zeros.)
      const int64_t v = v0 + row + 32 * q;
      w[stage][q].load(static_cast<const T*>(a.weight) + min(v, a.vocab - 1) * a.weight_ld,
                       c0 + chunk * 8, v < a.vocab ? a.width : 0);
    }
    if (with_d) {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
#pragma unroll
        for (int q = 0; q < kPiecesD; ++q) {
          d[stage][p][q] = *reinterpret_cast<const u32x4_t*>(
              a.d + p * a.d_plane + (row + 32 * q) * a.d_ld + v0 + chunk * 8);
        }
      }
    }
  };
  f32x4_t acc[N];
#pragma unroll
  for (int n = 0; n < N; ++n) acc[n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto round = [&](int s, int64_t t) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 2; ++q) w[s][q].store(weight[s] + place_w + q * 32 * 64, kPlaneW);
    if (with_d) {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
#pragma unroll
        for (int q = 0; q < kPiecesD; ++q) {
          *reinterpret_cast<u32x4_t*>(ds[s] + p * kPlaneD + place_d + q * 32 * 64) = d[s][p][q];
        }
      }
    }
    load(s, t + 2);
    // One barrier a round: a buffer is written again behind the next one's.
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8_t fw[kPlanes], fd[kParts][N];
#pragma unroll
      for (int p = 0; p < kPlanes; ++p) {
        const uint16_t* from = weight[s] + p * kPlaneW + (h * 32 + g * 8 + (l >> 2)) * 64 +
                               ((2 * wave + ((l & 3) >> 1)) ^ ((l >> 2) << 1)) * 8 + (l & 1) * 4;
        const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)from);
        const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(from + 4 * 64));
        fw[p] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
      }
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          fd[p][n] = *reinterpret_cast<const bf16x8_t*>(
              ds[s] + p * kPlaneD + (n * 16 + l) * 64 + (((h * 4 + g) ^ (l & 7)) * 8));
        }
      }
#pragma unroll
      for (int pass = 0; pass < kThinPasses<T>; ++pass) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              fw[thin_a_part<T>(pass)], fd[thin_d_part<T>(pass)][n], acc[n], 0, 0, 0);
        }
      }
    }
  };
  if (begin < end) {
    load(0, begin);
    load(1, begin + 1);
  }
  for (int64_t t = begin; t < end; t += 2) {
    round(0, t);
    if (t + 1 >= end) break;
    round(1, t + 1);
  }
  const int i = c0 + wave * 16 + g * 4;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int j = n * 16 + l;
    if (j >= count || i >= a.width) continue;
    f32x4_t* sum = reinterpret_cast<f32x4_t*>(
        a.sum + (static_cast<int64_t>(blockIdx.y) * kThinRows + j) * a.sum_ld + i);
    *sum = a.load_sum ? acc[n] + *sum : acc[n];
  }
}

// dweight of no rows, as 16-bit values.
__global__ __launch_bounds__(256) void zero_weight(uint16_t* out, int64_t n) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256 * 8;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n; i += step) {
    if (i + 8 <= n) {
      *reinterpret_cast<u32x4_a2_t*>(out + i) = u32x4_t{0u, 0u, 0u, 0u};
    } else {
      for (int64_t m = i; m < n; ++m) out[m] = 0;
    }
  }
}

// One workgroup a row.
__global__ __launch_bounds__(256) void join_thin(Thin a, int64_t ignore_index, float* loss,
                                                 float* lse) {
  __shared__ float2 parts[4];
  const int j = blockIdx.x;
  const int64_t tok = token_at(a.tokens, a.token_size, j);
  if (tok == ignore_index) {
    if (threadIdx.x == 0) loss[j] = lse[j] = 0.0f;
    return;
  }
  float top = -kLargest, sum = 0.0f;
#pragma unroll 4
  for (int64_t t = threadIdx.x; t < a.tiles; t += 256) join_one(top, sum, a.part[j * a.tiles + t]);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    join_one(top, sum, make_float2(__shfl_xor(top, o), __shfl_xor(sum, o)));
  }
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int q = 1; q < 4; ++q) join_one(top, sum, parts[q]);
    const bool known = tok >= 0 && tok < a.vocab;
    put_loss(top, sum, known ? a.target[j] : __builtin_nanf(""), loss + j, lse + j);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

inline int64_t tiles_of(int64_t rows_a, int64_t rows_b, int tile) {
  return (up(rows_a, tile) / tile) * (up(rows_b, tile) / tile);
}

// Where things lie in the workspace; pieces of the vocabulary are multiples of
// kTile rows and of one size.
struct Plan {
  int64_t rows_pad, sum_rows, k_pad, piece, pieces;
  int planes, d_planes;
  int tile, tile_hidden, tile_weight;  // of the logits, dhidden and dweight
  int splits;                          // of a piece, for dhidden
  bool direct;                         // weight is read where it lies
  bool thin;                           // few rows: the kernels of their own,
  bool thin_gemm;                      // but for dhidden of aligned bf16
  bool two_parts;                      // of bf16 operands' d, of more rows
  size_t kept, count, target, part, hidden, weight, d, sum, bytes;
};

constexpr int64_t kMostTiles = int64_t{1} << 22;  // 2^31 threads
constexpr int64_t kMostRows = (int64_t{1} << 22) - kTile;  // a tile's bytes fit 31 bits
constexpr size_t kForwardBytes = size_t{1024} << 20;  // of a copied piece
constexpr size_t kBackwardBytes = size_t{1536} << 20;  // of a piece's d and copies

// The tile with which a product ends sooner.  256 large tiles run at once (one a
// CU, for its LDS), or 512 small ones; a round of all takes about 1.5 us, or 1.0
// (for two thirds of the LDS reads at half the products), and what is around the
// rounds of a tile about 12 us, or 7.  Measured, large and small: 4096 x 1024 x
// 32000 (2000 tiles) 304 and 389 us, 512 x 2048 x 8000 (64 tiles) 48 and 28 us.
struct Work {
  int64_t tiles, rounds;
};

int64_t time_of(Work w, int tile) {
  const int64_t at_once = tile == kTile ? kCus : 2 * kCus;
  const int64_t waves = (w.tiles + at_once - 1) / at_once;
  return waves * (tile == kTile ? 15 * w.rounds + 120 : 10 * w.rounds + 70);
}

template <typename WorkOf>
int better_tile(WorkOf work_of) {
  return time_of(work_of(kTile), kTile) <= time_of(work_of(kSmallTile), kSmallTile) ? kTile
                                                                                    : kSmallTile;
}

Plan plan_of(const void* weight, int elem_size, int64_t rows, int64_t width, int64_t vocab,
             int64_t weight_ld, bool backward, bool two_parts) {
  Plan p{};
  if (!backward && rows <= kThinRows) {
    p.target = 0;
    p.part = up(sizeof(float) * rows, 256);
    p.bytes = p.part + sizeof(float2) * rows * (up(vocab, kThinTile) / kThinTile);
    return p;
  }
  p.planes = elem_size == 2 ? 1 : 3;
  const bool aligned = elem_size == 2 && aligned16(weight) && weight_ld % 8 == 0 && width % 8 == 0;
  p.thin = rows <= kThinRows;
  p.thin_gemm = p.thin && aligned;
  p.direct = p.thin || aligned;
  p.rows_pad = p.thin ? kThinRows : up(rows, kTile);
  p.two_parts = two_parts && elem_size == 2 && !p.thin;
  p.d_planes = (p.thin && elem_size == 2) || p.two_parts ? 2 : p.planes;
  p.sum_rows = p.thin_gemm ? 2 * kThinRows : p.rows_pad;
  p.k_pad = up(width, kStep);
  const size_t copy = p.direct ? 0 : sizeof(uint16_t) * p.planes * p.k_pad;
  const size_t per_row =
      backward ? copy + sizeof(uint16_t) * p.d_planes * p.rows_pad : copy;
  const size_t most = backward ? kBackwardBytes : kForwardBytes;
  const int64_t whole = up(vocab, kTile);
  int64_t piece = whole;
  if (per_row > 0) {
    piece = std::min<int64_t>(whole, std::max<int64_t>(kTile, most / per_row / kTile * kTile));
  }
  piece = std::min(piece, kMostRows);  // a row of d
  // Tiles of one launch.
  const int64_t other = std::max(p.rows_pad, up(width, kTile)) / kTile;
  piece = std::min(piece, std::max<int64_t>(1, kMostTiles / other) * kTile);
  p.pieces = (vocab + piece - 1) / piece;
  p.piece = up((vocab + p.pieces - 1) / p.pieces, kTile);
  p.pieces = (vocab + p.piece - 1) / p.piece;
  const int64_t passes = elem_size == 2 ? 1 : 6, in_piece = std::min(p.piece, vocab);
  const int64_t passes_d = p.two_parts ? 2 : passes;
  p.tile = better_tile([&](int tile) {
    return Work{tiles_of(in_piece, rows, tile), passes * p.k_pad / kStep};
  });
  p.tile_weight = better_tile([&](int tile) {
    return Work{tiles_of(width, in_piece, tile), passes_d * up(rows, kStep) / kStep};
  });
  // dhidden has few tiles where there are few rows: the piece is split until
  // there are as many workgroups as run at once, 8 rounds each at least.
  auto splits_of = [&](int tile) {
    const int64_t at_once = tile == kTile ? kCus : 2 * kCus;
    return std::max<int64_t>(1, std::min(at_once / tiles_of(width, p.sum_rows, tile),
                                         p.piece / (8 * kStep)));
  };
  p.tile_hidden = better_tile([&](int tile) {
    const int64_t splits = splits_of(tile);
    return Work{splits * tiles_of(width, p.sum_rows, tile), passes_d * p.piece / kStep / splits};
  });
  p.splits = static_cast<int>(splits_of(p.tile_hidden));
  if (p.thin && !p.thin_gemm) {
    // Several workgroups a CU, of 2 rounds at least, and not too many to join.
    p.splits = static_cast<int>(std::max<int64_t>(
        1, std::min({2048 / (up(width, 64) / 64), int64_t{128}, in_piece / 128})));
  }
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += up(bytes, 256);
    return here;
  };
  const size_t plane = sizeof(uint16_t) * p.planes;
  p.kept = take(sizeof(int) * rows);
  p.count = take(sizeof(int));
  p.hidden = take(plane * p.rows_pad * p.k_pad);
  p.weight = take(p.direct ? 0 : plane * p.piece * p.k_pad);
  if (backward) {
    p.d = take(sizeof(uint16_t) * p.d_planes * p.rows_pad * p.piece);
    p.sum = take(p.thin || p.pieces * p.splits > 1
                     ? sizeof(float) * p.splits * p.sum_rows * up(width, 4) : 0);
  } else {
    p.target = take(sizeof(float) * rows);
    p.part = take(sizeof(float2) * (up(vocab, p.tile) / p.tile) * p.rows_pad);
  }
  p.bytes = at;
  return p;
}

bool sizes_fit(int64_t rows, int64_t width, int64_t vocab, int64_t hidden_ld, int64_t weight_ld) {
  return rows >= 0 && rows <= kMostRows && vocab >= 1 &&
         vocab <= (int64_t{1} << 31) - 65536 && width >= 1 && width <= (1 << 20) &&
         hidden_ld >= width && weight_ld >= width && weight_ld <= (1 << 21) &&
         up(rows, kTile) / kTile * (up(width, kTile) / kTile) <= kMostTiles;
}

int check_operands(const char* what, int elem_size, int token_size, int64_t rows, int64_t width,
                   int64_t vocab, int64_t hidden_ld, int64_t weight_ld, float scale) {
  HIPO_REQUIRE(elem_size == 2 || elem_size == 4, "%s: elem_size must be 2 or 4", what);
  HIPO_REQUIRE(token_size == 4 || token_size == 8, "%s: token_size must be 4 or 8", what);
  HIPO_REQUIRE(rows >= 0 && width >= 0 && vocab >= 0, "%s: negative size", what);
  HIPO_REQUIRE(width >= 1 && width <= (1 << 20), "%s: width must be from 1 to 2^20", what);
  HIPO_REQUIRE(vocab >= 1, "%s: empty vocabulary", what);
  HIPO_REQUIRE(hidden_ld >= width && weight_ld >= width, "%s: row_stride below width", what);
  HIPO_REQUIRE(sizes_fit(rows, width, vocab, hidden_ld, weight_ld),
               "%s: at most 2^22 - 256 rows, a vocabulary of 2^31 - 65536, a weight_row_stride of "
               "2^21 and rows * width of 2^38", what);
  HIPO_REQUIRE(scale >= 0x1p-100f && scale <= 0x1p100f,
               "%s: scale must be from 2^-100 to 2^100", what);
  return 0;
}

template <typename T>
int pack(const char* what, Pack a, int64_t rows, hipStream_t stream) {
  pack_rows<T><<<static_cast<uint32_t>(std::min<int64_t>(rows, 1 << 16)), 256, 0, stream>>>(a);
  return check_launch(what);
}

template <typename T, Epilogue E, int Parts = sizeof(T) == 2 ? 1 : 3>
int multiply(const char* what, const Product& p, int tile, int64_t rows_b, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(tiles_of(p.a_rows, rows_b, tile) * p.splits);
  if (tile == kTile) {
    gemm<T, kTile, E, Parts><<<grid, 2 * kTile, 0, stream>>>(p);
  } else {
    gemm<T, kSmallTile, E, Parts><<<grid, 2 * kSmallTile, 0, stream>>>(p);
  }
  return check_launch(what);
}

// Of d, in one part or two where the operands are bf16.
template <typename T, Epilogue E>
int multiply_d(const char* what, const Product& p, int tile, int64_t rows_b, bool two_parts,
               hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (two_parts) return multiply<T, E, 2>(what, p, tile, rows_b, stream);
  }
  return multiply<T, E>(what, p, tile, rows_b, stream);
}

struct Call {
  const void *hidden, *weight, *tokens;
  int token_size;
  int64_t rows, width, vocab, hidden_ld, weight_ld;
  float scale;
  int64_t ignore_index;
  char* ws;
  hipStream_t stream;

  template <typename P>
  P* at(size_t offset) const {
    return reinterpret_cast<P*>(ws + offset);
  }
};

#define HIPO_STEP(call)              \
  do {                               \
    const int step_rc = (call);      \
    if (step_rc != 0) return step_rc; \
  } while (0)

// The operands of a piece's logits: the vocabulary's rows from `first` on.
template <typename T>
int piece_of_weight(const char* what, const Call& c, const Plan& plan, int64_t first, Product* g) {
  g->a_rows = static_cast<int>(std::min(plan.piece, c.vocab - first));
  const T* from = static_cast<const T*>(c.weight) + first * c.weight_ld;
  if (plan.direct) {  // (of few rows at any alignment: gemm() does not read it)
    g->a = reinterpret_cast<const uint16_t*>(from);
    g->lda = c.weight_ld;
    g->k = static_cast<int>(c.width);
  } else {
    uint16_t* to = c.at<uint16_t>(plan.weight);
    g->a = to;
    g->lda = plan.k_pad;
    g->a_plane = plan.piece * plan.k_pad;
    g->k = static_cast<int>(plan.k_pad);
    const Pack all{from, c.weight_ld, nullptr, nullptr, g->a_rows, static_cast<int>(c.width),
                   to, plan.k_pad, g->a_plane, nullptr, 0, 0, nullptr};
    HIPO_STEP(pack<T>(what, all, g->a_rows, c.stream));
  }
  g->first = first;
  return 0;
}

template <typename T>
int select_and_pack(const char* what, const Call& c, const Plan& plan, float* loss, float* lse,
                    void* dhidden, Product* g) {
  int* kept = c.at<int>(plan.kept);
  int* count = c.at<int>(plan.count);
  float* target = loss ? c.at<float>(plan.target) : nullptr;
  uint16_t* hidden = c.at<uint16_t>(plan.hidden);
  const int64_t plane = plan.rows_pad * plan.k_pad;
  const Select select{c.tokens, c.token_size, c.rows, c.ignore_index, kept, count, target, loss,
                      lse};
  const Pack rows{c.hidden, c.hidden_ld, kept, count, c.rows, static_cast<int>(c.width), hidden,
                  plan.k_pad, plane, c.tokens, c.token_size, c.ignore_index, dhidden};
  if (c.rows <= kSelectRows) {
    select_and_pack_rows<T><<<static_cast<uint32_t>(c.rows), 256, 0, c.stream>>>(select, rows);
    HIPO_STEP(check_launch(what));
  } else {
    select_rows<<<1, 1024, 0, c.stream>>>(select);
    HIPO_STEP(check_launch(what));
    HIPO_STEP(pack<T>(what, rows, c.rows, c.stream));
  }
  g->b = hidden;
  g->ldb = plan.k_pad;
  g->b_plane = plane;
  g->b_count = count;
  g->tokens = c.tokens;
  g->token_size = c.token_size;
  g->kept = kept;
  g->splits = 1;
  g->scale = c.scale;
  g->vocab = c.vocab;
  g->target = target;
  return 0;
}

template <typename T, bool Grad>
int launch_thin(const char* what, const Thin& a, int64_t rows, hipStream_t stream) {
  const uint32_t grid = static_cast<uint32_t>(std::min<int64_t>(a.tiles, 1 << 20));
  // No more workgroups than CUs: K split, as far as LDS and registers reach (4 x
  // 3584 x 3968 bf16, 62 workgroups: 22.1 -> 15.2 us; 1 x 2048 x 32000, 500
  // workgroups: 23.9 -> 30.5, so not there).  Four groups leave a lane 128 registers:
  // of 17 to 32 rows the forward spills with them (24 x 2048 x 16000: 22.2 us, two
  // groups 19.5; 32 x 3584 x 3968: 21.0, 20.9), the gradient does not (24 x 2048 x
  // 16000: 67.4, 66.4; 32 x 4096 x 8000: 62.6, 63.9).
  const bool few = a.tiles <= kCus;
  constexpr int kMany = sizeof(T) == 2 ? 4 : 2, kWide = sizeof(T) == 2 ? 2 : 1;
  constexpr int kMiddle = Grad ? kMany : 2;
  // Rows that are whole 128-byte lines, read once: past the caches, which hold other
  // layers' weights by the next call (1 x 4096 x 128000 203 -> 187 us, 1 x 2048 x 32000
  // among other states 37.8 -> 33.9; the same 131 MB at once again 26.8 -> 32.0).  Of
  // other rows (3 x 1000 x 20001) 17.4 -> 20.3, as two rows' reads meet in a line; the
  // gradient reads the weight twice (8 x 2048 x 32000 117 -> 119).
  constexpr bool kOnce = sizeof(T) == 2 && !Grad;
  const bool once = kOnce && reinterpret_cast<uintptr_t>(a.weight) % 128 == 0 &&
                    a.weight_ld % 64 == 0;
  if (rows <= 16) {
    few    ? thin_logits<T, 1, Grad, kMany><<<grid, 256 * kMany, 0, stream>>>(a)
    : once ? thin_logits<T, 1, Grad, 1, kOnce><<<grid, 256, 0, stream>>>(a)
           : thin_logits<T, 1, Grad, 1><<<grid, 256, 0, stream>>>(a);
  } else if (rows <= 32) {
    few    ? thin_logits<T, 2, Grad, kMiddle><<<grid, 256 * kMiddle, 0, stream>>>(a)
    : once ? thin_logits<T, 2, Grad, 1, kOnce><<<grid, 256, 0, stream>>>(a)
           : thin_logits<T, 2, Grad, 1><<<grid, 256, 0, stream>>>(a);
  } else {
    few    ? thin_logits<T, 4, Grad, kWide><<<grid, 256 * kWide, 0, stream>>>(a)
    : once ? thin_logits<T, 4, Grad, 1, kOnce><<<grid, 256, 0, stream>>>(a)
           : thin_logits<T, 4, Grad, 1><<<grid, 256, 0, stream>>>(a);
  }
  return check_launch(what);
}

template <typename T>
int run_thin(const Call& c, const Plan& plan, float* loss, float* lse) {
  const char* what = "linear_cross_entropy";
  const Thin a{c.hidden,    c.weight,    c.tokens, c.token_size, static_cast<int>(c.rows),
               static_cast<int>(c.width), c.vocab, c.hidden_ld,  c.weight_ld,
               c.scale,     c.at<float2>(plan.part), c.at<float>(plan.target),
               up(c.vocab, kThinTile) / kThinTile};
  HIPO_STEP((launch_thin<T, false>(what, a, c.rows, c.stream)));
  join_thin<<<static_cast<uint32_t>(c.rows), 256, 0, c.stream>>>(a, c.ignore_index, loss, lse);
  return check_launch(what);
}

template <typename T>
int run_fwd(const Call& c, const Plan& plan, float* loss, float* lse) {
  const char* what = "linear_cross_entropy";
  if (c.rows <= kThinRows) return run_thin<T>(c, plan, loss, lse);
  Product g{};
  HIPO_STEP(select_and_pack<T>(what, c, plan, loss, lse, nullptr, &g));
  g.part = c.at<float2>(plan.part);
  g.part_ld = plan.rows_pad;
  for (int64_t i = 0; i < plan.pieces; ++i) {
    HIPO_STEP(piece_of_weight<T>(what, c, plan, i * plan.piece, &g));
    g.first_tile = i * plan.piece / plan.tile;
    HIPO_STEP((multiply<T, kReduce>(what, g, plan.tile, c.rows, c.stream)));
  }
  const int tiles = static_cast<int>(up(c.vocab, plan.tile) / plan.tile);
  join_loss<<<static_cast<uint32_t>(std::min<int64_t>((c.rows + 15) / 16, 1 << 16)), 256, 0,
              c.stream>>>(
      JoinLoss{g.part, g.part_ld, tiles, g.kept, g.b_count, g.target, loss, lse});
  return check_launch(what);
}

template <typename T>
int run_bwd(const char* what, const Call& c, const Plan& plan, const float* grad,
            const float* lse, const float* grad_lse, void* dhidden, void* dweight) {
  Product g{};
  HIPO_STEP(select_and_pack<T>(what, c, plan, nullptr, nullptr, dhidden, &g));
  const int width = static_cast<int>(c.width);
  g.grad = grad;
  g.lse = lse;
  g.grad_lse = grad_lse;
  g.d = c.at<uint16_t>(plan.d);
  g.d_ld = plan.piece;
  g.d_plane = plan.rows_pad * plan.piece;
  for (int64_t i = 0; i < plan.pieces; ++i) {
    const int64_t first = i * plan.piece;
    HIPO_STEP(piece_of_weight<T>(what, c, plan, first, &g));
    if (plan.thin) {
      Thin t{};
      t.hidden = c.hidden;
      t.weight = static_cast<const T*>(c.weight) + first * c.weight_ld;
      t.tokens = c.tokens;
      t.token_size = c.token_size;
      t.width = width;
      t.vocab = g.a_rows;
      t.hidden_ld = c.hidden_ld;
      t.weight_ld = c.weight_ld;
      t.scale = c.scale;
      t.tiles = up(g.a_rows, kThinTile) / kThinTile;
      t.kept = g.kept;
      t.count = g.b_count;
      t.grad = grad;
      t.lse = lse;
      t.grad_lse = grad_lse;
      t.d = g.d;
      t.d_ld = g.d_ld;
      t.d_plane = g.d_plane;
      t.first = first;
      t.whole_vocab = c.vocab;
      HIPO_STEP((launch_thin<T, true>(what, t, c.rows, c.stream)));
      if (plan.thin_gemm) {
        // d's two parts as 128 rows, whose sums join_hidden() adds.
        Product h{};
        h.a = g.a;
        h.lda = g.lda;
        h.a_rows = width;
        h.a_k = g.a_rows;
        h.b = g.d;
        h.ldb = g.d_ld;
        h.b_rows = 2 * kThinRows;
        h.k = static_cast<int>(up(g.a_rows, kStep));
        h.splits = plan.splits;
        h.sum = c.at<float>(plan.sum);
        h.sum_ld = up(c.width, 4);
        h.sum_plane = plan.sum_rows * h.sum_ld;
        h.load_sum = i > 0;
        HIPO_STEP((multiply<T, kAccumulate>(what, h, plan.tile_hidden, h.b_rows, c.stream)));
      } else {
        const ThinHidden h{t.weight, c.weight_ld, g.a_rows, width, g.d, g.d_ld, g.d_plane,
                           g.b_count, c.at<float>(plan.sum), up(c.width, 4), i > 0};
        const dim3 grid(static_cast<uint32_t>(up(c.width, 64) / 64), plan.splits);
        if (c.rows <= 16) {
          thin_hidden<T, 1><<<grid, 256, 0, c.stream>>>(h);
        } else if (c.rows <= 32) {
          thin_hidden<T, 2><<<grid, 256, 0, c.stream>>>(h);
        } else {
          thin_hidden<T, 4><<<grid, 256, 0, c.stream>>>(h);
        }
        HIPO_STEP(check_launch(what));
      }
      // Columns in as many parts as it takes to fill the CUs several times.
      const int64_t strips = up(g.a_rows, 64) / 64, all = up(c.width, 64) / 64;
      const int64_t parts = std::min<int64_t>(all, std::max<int64_t>(1, 2048 / strips));
      const int chunks = static_cast<int>((all + parts - 1) / parts);
      thin_weight<T><<<dim3(static_cast<uint32_t>(strips),
                            static_cast<uint32_t>((all + chunks - 1) / chunks)),
                       256, 0, c.stream>>>(
          ThinWeight{g.b, g.d, g.ldb, g.b_plane, g.d_ld, g.d_plane, g.b_count, width, g.a_rows,
                     static_cast<T*>(dweight) + first * c.width, c.width, chunks});
      HIPO_STEP(check_launch(what));
      continue;
    }
    HIPO_STEP((multiply_d<T, kLogitGrad>(what, g, plan.tile, c.rows, plan.two_parts, c.stream)));

    Product h{};
    h.a = g.a;
    h.lda = g.lda;
    h.a_plane = g.a_plane;
    h.a_rows = width;
    h.a_k = g.a_rows;
    h.b = g.d;
    h.ldb = g.d_ld;
    h.b_plane = g.d_plane;
    h.b_count = g.b_count;
    h.k = static_cast<int>(up(g.a_rows, kStep));
    h.kept = g.kept;
    h.sum = c.at<float>(plan.sum);
    h.sum_ld = up(c.width, 4);
    h.sum_plane = plan.rows_pad * h.sum_ld;
    h.splits = plan.splits;
    h.load_sum = i > 0;
    h.to_out = plan.splits == 1 && i + 1 == plan.pieces;
    h.out = dhidden;
    h.out_ld = c.width;
    HIPO_STEP((multiply_d<T, kAccumulate>(what, h, plan.tile_hidden, c.rows, plan.two_parts,
                                          c.stream)));

    Product w{};
    w.a = g.b;
    w.lda = g.ldb;
    w.a_plane = g.b_plane;
    w.a_rows = width;
    w.b = g.d;
    w.ldb = g.d_ld;
    w.b_plane = g.d_plane;
    w.b_rows = g.a_rows;
    w.k_count = g.b_count;
    w.splits = 1;
    w.out = static_cast<T*>(dweight) + first * c.width;
    w.out_ld = c.width;
    HIPO_STEP((multiply_d<T, kStore>(what, w, plan.tile_weight, g.a_rows, plan.two_parts,
                                     c.stream)));
  }
  if (plan.thin || plan.splits > 1) {
    const int64_t blocks = (c.rows * ((c.width + 3) / 4) + 255) / 256;
    join_hidden<T><<<static_cast<uint32_t>(std::min<int64_t>(blocks, 1 << 16)), 256, 0,
                     c.stream>>>(c.at<float>(plan.sum), up(c.width, 4),
                                 plan.sum_rows * up(c.width, 4), plan.splits, plan.thin_gemm,
                                 g.kept, g.b_count, static_cast<T*>(dhidden), width);
    return check_launch(what);
  }
  return 0;
}

}  // namespace
}  // namespace hipo

extern "C" size_t hipo_linear_cross_entropy_workspace_bytes(const void* weight, int elem_size,
                                                            int64_t rows, int64_t width,
                                                            int64_t vocab,
                                                            int64_t weight_row_stride) {
  if ((elem_size != 2 && elem_size != 4) || rows == 0 ||
      !hipo::sizes_fit(rows, width, vocab, width, weight_row_stride)) {
    return 0;
  }
  return hipo::plan_of(weight, elem_size, rows, width, vocab, weight_row_stride, false, false)
      .bytes;
}

extern "C" int hipo_linear_cross_entropy(const void* hidden, const void* weight, int elem_size,
                                         const void* tokens, int token_size, float* loss,
                                         float* lse, int64_t rows, int64_t width, int64_t vocab,
                                         int64_t hidden_row_stride, int64_t weight_row_stride,
                                         float scale, int64_t ignore_index, void* workspace,
                                         size_t workspace_bytes, hipStream_t stream) {
  using namespace hipo;
  clear_error();
  const char* what = "linear_cross_entropy";
  HIPO_STEP(check_operands(what, elem_size, token_size, rows, width, vocab, hidden_row_stride,
                           weight_row_stride, scale));
  if (rows == 0) return 0;
  HIPO_REQUIRE(hidden && weight && tokens && loss && lse, "%s: null pointer", what);
  const Plan plan = plan_of(weight, elem_size, rows, width, vocab, weight_row_stride, false,
                            false);
  HIPO_REQUIRE(workspace && workspace_bytes >= plan.bytes && aligned16(workspace),
               "%s: workspace of %zu bytes, 16-byte aligned, needed", what, plan.bytes);
  const Call c{hidden, weight, tokens, token_size, rows, width, vocab, hidden_row_stride,
               weight_row_stride, scale, ignore_index, static_cast<char*>(workspace), stream};
  return elem_size == 2 ? run_fwd<uint16_t>(c, plan, loss, lse)
                        : run_fwd<float>(c, plan, loss, lse);
}

namespace hipo {
namespace {

size_t bwd_workspace_bytes(const void* weight, int elem_size, int64_t rows, int64_t width,
                           int64_t vocab, int64_t weight_ld, bool two_parts) {
  if ((elem_size != 2 && elem_size != 4) || rows == 0 ||
      !sizes_fit(rows, width, vocab, width, weight_ld)) {
    return 0;
  }
  return plan_of(weight, elem_size, rows, width, vocab, weight_ld, true, two_parts).bytes;
}

int bwd(const char* what, const float* grad, int elem_size, const float* lse,
        const float* grad_lse, void* dhidden, void* dweight, const Call& c,
        size_t workspace_bytes, bool two_parts) {
  clear_error();
  HIPO_STEP(check_operands(what, elem_size, c.token_size, c.rows, c.width, c.vocab, c.hidden_ld,
                           c.weight_ld, c.scale));
  if (c.rows == 0) {
    if (!dweight) return 0;
    const int64_t n = c.vocab * c.width * (elem_size / 2);
    zero_weight<<<static_cast<uint32_t>(std::min<int64_t>(up(n, 2048) / 2048, 1 << 16)), 256, 0,
                  c.stream>>>(static_cast<uint16_t*>(dweight), n);
    return check_launch(what);
  }
  HIPO_REQUIRE(grad && c.hidden && c.weight && c.tokens && lse && dhidden && dweight,
               "%s: null pointer", what);
  const Plan plan = plan_of(c.weight, elem_size, c.rows, c.width, c.vocab, c.weight_ld, true,
                            two_parts);
  HIPO_REQUIRE(c.ws && workspace_bytes >= plan.bytes && aligned16(c.ws),
               "%s: workspace of %zu bytes, 16-byte aligned, needed", what, plan.bytes);
  return elem_size == 2
             ? run_bwd<uint16_t>(what, c, plan, grad, lse, grad_lse, dhidden, dweight)
             : run_bwd<float>(what, c, plan, grad, lse, grad_lse, dhidden, dweight);
}

}  // namespace
}  // namespace hipo

extern "C" size_t hipo_linear_cross_entropy_bwd_workspace_bytes(
    const void* weight, int elem_size, int64_t rows, int64_t width, int64_t vocab,
    int64_t weight_row_stride) {
  return hipo::bwd_workspace_bytes(weight, elem_size, rows, width, vocab, weight_row_stride,
                                   false);
}

extern "C" int hipo_linear_cross_entropy_bwd(const float* grad, const void* hidden,
                                             const void* weight, int elem_size,
                                             const void* tokens, int token_size, const float* lse,
                                             const float* grad_lse, void* dhidden, void* dweight,
                                             int64_t rows, int64_t width, int64_t vocab,
                                             int64_t hidden_row_stride, int64_t weight_row_stride,
                                             float scale, int64_t ignore_index, void* workspace,
                                             size_t workspace_bytes, hipStream_t stream) {
  return hipo::bwd("linear_cross_entropy_bwd", grad, elem_size, lse, grad_lse, dhidden, dweight,
                   {hidden, weight, tokens, token_size, rows, width, vocab, hidden_row_stride,
                    weight_row_stride, scale, ignore_index, static_cast<char*>(workspace), stream},
                   workspace_bytes, false);
}

extern "C" size_t hipo_linear_cross_entropy_bwd_two_parts_workspace_bytes(
    const void* weight, int elem_size, int64_t rows, int64_t width, int64_t vocab,
    int64_t weight_row_stride) {
  return hipo::bwd_workspace_bytes(weight, elem_size, rows, width, vocab, weight_row_stride,
                                   true);
}

extern "C" int hipo_linear_cross_entropy_bwd_two_parts(
    const float* grad, const void* hidden, const void* weight, int elem_size,
    const void* tokens, int token_size, const float* lse, const float* grad_lse, void* dhidden,
    void* dweight, int64_t rows, int64_t width, int64_t vocab, int64_t hidden_row_stride,
    int64_t weight_row_stride, float scale, int64_t ignore_index, void* workspace,
    size_t workspace_bytes, hipStream_t stream) {
  return hipo::bwd("linear_cross_entropy_bwd_two_parts", grad, elem_size, lse, grad_lse, dhidden,
                   dweight,
                   {hidden, weight, tokens, token_size, rows, width, vocab, hidden_row_stride,
                    weight_row_stride, scale, ignore_index, static_cast<char*>(workspace), stream},
                   workspace_bytes, true);
}
