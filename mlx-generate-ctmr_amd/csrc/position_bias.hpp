// A learned bias of attention scores by the distance of a row and a key on each of
// up to four axes.
//
//   bias_ij = sum_a table[row_a(x_a(j) - x_a(i))][h]
// where x_a is a token's place on axis a, 0 .. extent_a - 1, and row_a the table's row
// for a distance (its bucket).  A workgroup lays the head's values out in LDS, the axes
// in two pairs: one value for each two distances of a pair, (2 e - 1) (2 e' - 1) of
// them, summed, in the scores' units.  Tokens have codes, places times strides, whose
// difference is the LDS address of both pairs' values: a score costs two subtractions, two
// reads and an addition, whatever the places and their order (without a cap the products
// are added to it by the matrix units).  The forward pass is bound by the latency of these
// reads: 2 x 16 heads of 64, 4096 rows on 16x16x16, bf16, 257 us where no bias takes 163:
// 4 LDS instructions where 1 was, and waves wait 2.5 times as long, three of them a SIMD,
// while no unit is full (LDS 37 % of the time, vector units 52, matrix units 21 for 38; no
// bank conflicts).  Heads of 32 187 us (116), of 128 358 (270).
//
// The table's gradient is the sum of the scores' gradients ds of a head over all pairs of
// a distance.  For a row i, ds_ij counts by the key's place on each axis, so with a
// column c = (a, x) for each place of each axis and one-hot rows o_j[a, x] = (x_a(j) == x)
//   dr_i[c] = sum_j ds_ij o_j[c]
// is a matrix product, which the matrix units sum without an addition in memory; the
// rows' dr are then added by distance.  o is exact in bf16 and the same for all heads: it
// streams through LDS beside the keys.  ds goes in three bf16 parts, all of fp32's bits, or
// two, 2^-17 of it, where the table has 16 bits (both kernels of the backward pass, heads of
// 64, 4096 rows: 815 us, 761).
//
// (The bias itself as a product too, of o_j and each row's r_i[c] = table[row_a(x - x_a(i))]
// in parts, has no reads of single values, but r takes 24 to 64 registers and the product
// as long as that of keys of as many values.  Forward, bf16, 4096 rows on 16x16x16, heads
// of 64 243 us and of 128 557, where reads take 255 and 361; 16 heads of 64, 8192 rows on
// 32x32x8, 874 and 489; a row over 13824 keys 66 and 52.  Tiles whose lanes share the reads
// of four keys in a line take 261 us for heads of 64, but 260 for 245 where keys are in no
// order and 294 for 192 with heads of 32: one form for all.)
#pragma once

#include "masked_attention.hpp"

namespace ctmr {
namespace attn {

constexpr int kColumns = 128;    // at most, over all axes
constexpr int kDistances = 256;  // numbers of distances: two for a place, and one to spare
constexpr int kAxes = 4;
constexpr int kMostValues = 8192;  // of both pairs: with 128 places on four axes 7938 at most

// A plan of places (ctmr_buckets), and the table.
struct Bias {
  const int* rows;                             // (kDistances) the table's row of a distance's number, -1 for none
  const unsigned *query_codes, *key_codes;     // (items, rows up to a multiple of kTile), of the axes in pairs
  const unsigned *query_places, *key_places;   // likewise: a byte for each axis
  const __bf16* key_hot;                       // (items, lk, 16 ST) o
  int64_t query_item, key_item, hot_item;      // from item to item in rows; 0: all have the same
  const void* table;                           // (table_rows, hq)
  int elem, table_rows, axes;
  int extents[kAxes], first_column[kAxes], first_number[kAxes];  // of each axis
  int pair_extents[kAxes], pair_number[kAxes];  // the axes in pairs, 0 and 1, 2 and 3; extent 1 and number -1: no axis
  int values;      // of both pairs
  unsigned reach;  // extent - 1 of each axis in its byte
  float* part;  // the gradient: (n, hq, slots, kDistances) sums over a block's rows, or null
  int slots;
};

// ST: contraction steps of 16 columns, 3, 4, 6 or 8, in the table's gradient; 0: no bias.
template <int ST>
struct BiasOf : Bias {};
template <>
struct BiasOf<0> {};

// A tile of one-hot rows in LDS: 64 columns, and 32 or 64 more behind them; zeros past 16 ST.
template <int ST>
struct HotTile {
  static constexpr int kBlocks = ST == 6 ? 3 : ST == 8 ? 4 : 2;  // of 32 columns
  static constexpr int kRow = 16 * ST;                           // columns of a row in memory
  static constexpr int kFirst = kTile * 128, kBytes = kTile * 64 * kBlocks;
  typedef Tile<__bf16, 64> First;
  typedef Tile<__bf16, ST == 6 ? 32 : 64> Second;

  // A operand whose rows are the columns 32 block .. + 31 (Tile::down).
  static __device__ __forceinline__ Frag<__bf16> down(const char* tile, int row, int block, int lane) {
    return block < 2 ? First::down(tile, row, block, lane) : Second::down(tile + kFirst, row, block - 2, lane);
  }
  // Rows from `first` of `count` straight into LDS.
  template <int THREADS>
  static __device__ __forceinline__ void load(char* tile, const __bf16* rows, int first, int count, int t) {
    Rows<__bf16, kTile> r;
    r.begin(rows, kRow, first, count, kRow < 64 ? kRow : 64);
    Stream<__bf16, 64, kTile, THREADS>::load(tile, r, t);
    if constexpr (ST > 4) {
      r.begin(rows + 64, kRow, first, count, kRow - 64);
      Stream<__bf16, ST == 6 ? 32 : 64, kTile, THREADS>::load(tile + kFirst, r, t);
    }
  }
};
// In the forward call and in dk and dv, which have no columns: a bias, and one with weights in two and three parts
// (fine_weights).
constexpr int kBias = 1, kFineBias = 2, kFinestBias = 3;

// Whether the table's gradient has more digits than two bf16 parts of each ds.
__device__ __forceinline__ bool wide_table(const Bias& b) { return b.elem == CTMR_ELEM_F32; }

// With fp32 heads of 128 LDS has no room for pairs: the axes are looked up one by one, in tables of 256 values, by the
// bytes of the difference of places.
template <typename T, int D>
constexpr bool kSingle = sizeof(T) == 4 && D == 128;

// What a row's word and a key's differ by says where their values are.  Every lane has one: past the end that of the last.
template <bool SINGLE>
__device__ __forceinline__ unsigned row_word(const Bias& b, int item, int i, int lq) {
  const int64_t at = item * b.query_item + min(i, lq - 1);
  return SINGLE ? b.query_places[at] + b.reach : b.query_codes[at];
}
template <bool SINGLE>
__device__ __forceinline__ unsigned key_word(const Bias& b, int item, int j, int lk) {
  const int64_t at = item * b.key_item + min(j, lk - 1);
  return SINGLE ? b.key_places[at] : b.key_codes[at];
}

// Lays out head h's values in `values`, in units of 1 / `unit`, by all threads of the workgroup between its barriers.  A
// value below -2^100 hides a pair: the score that it makes is below kNone in log2 units (the host keeps the units so), also
// where several are summed.
template <bool SINGLE, int THREADS>
__device__ __forceinline__ void lay_out_bias(const Bias& b, char* values, int h, int hq, float unit, int t) {
  __shared__ float of[kDistances];
  for (int n = t; n < kDistances; n += THREADS) {
    const int row = b.rows[n];
    const float v = row < 0 ? 0.f : load_param(b.table, b.elem, (int64_t)row * hq + h);
    of[n] = v < -0x1p100f ? -0x1p127f : v * unit;
  }
  __syncthreads();
  float* out = reinterpret_cast<float*>(values);
  // Words count from the key to the row, numbers from the row to the key.
  if constexpr (SINGLE) {
#pragma unroll
    for (int a = 0; a < kAxes; ++a)
      for (int i = t; i < 256; i += THREADS)
        out[256 * a + i] = a < b.axes && i < 2 * b.extents[a] - 1 ? of[b.first_number[a] + 2 * b.extents[a] - 2 - i] : 0.f;
  } else {
#pragma unroll
    for (int p = 0; p < kAxes; p += 2) {
      const int n0 = 2 * b.pair_extents[p] - 1, n1 = 2 * b.pair_extents[p + 1] - 1;
      const int at0 = b.pair_number[p], at1 = b.pair_number[p + 1];
      for (int i = t; i < n0 * n1; i += THREADS) {
        const int x0 = i / n1, x1 = i - x0 * n1;
        out[i] = (at0 < 0 ? 0.f : of[at0 + n0 - 1 - x0]) + (at1 < 0 ? 0.f : of[at1 + n1 - 1 - x1]);
      }
      out += n0 * n1;
    }
  }
}

// Rows whose reads apply_bias has on their way at once, 32 registers for 16: heads of 128 have none to spare.
template <int D>
constexpr int kBiasRows = D == 128 ? 4 : 16;

// The bias of a lane's 16 scores, whose rows have `words` (32 of them, in LDS), or that added to the scores.  KEYS: the rows
// are keys.  Pairs: the lane's own two addresses less the halves of a word; else single axes, by the difference's bytes.
template <bool SINGLE, bool KEYS, bool ADD, int ROWS>
__device__ __forceinline__ void apply_bias(f16v& s, const char* values, unsigned own, const unsigned* words, int lane) {
  typedef __attribute__((address_space(3))) const char lds_char;
  typedef __attribute__((address_space(3))) const float lds_float;
  const unsigned base = (unsigned)(uintptr_t)(lds_char*)values;
  const auto value = [](unsigned at) { return *(lds_float*)(uintptr_t)at; };
  const unsigned own0 = KEYS ? base + (own & 0xffffu) : base - (own & 0xffffu);
  const unsigned own1 = KEYS ? base + (own >> 16) : base - (own >> 16);
#pragma unroll
  for (int g = 0; g < 16; g += ROWS) {
    unsigned w[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r += 4) {
      const u4 v = *reinterpret_cast<const u4*>(words + 2 * (g + r) + 4 * (lane >> 5));
#pragma unroll
      for (int e = 0; e < 4; ++e) w[r + e] = v[e];
    }
    float first[ROWS], second[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if constexpr (SINGLE) {
        const unsigned at = KEYS ? own - w[r] : w[r] - own;
        first[r] = value(base + (at & 255u) * 4) + value(base + 1024 + (at >> 8 & 255u) * 4);
        second[r] = value(base + 2048 + (at >> 16 & 255u) * 4) + value(base + 3072 + (at >> 24) * 4);
      } else {
        first[r] = value(KEYS ? own0 - (w[r] & 0xffffu) : own0 + (w[r] & 0xffffu));
        second[r] = value(KEYS ? own1 - (w[r] >> 16) : own1 + (w[r] >> 16));
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[g + r] = (ADD ? s[g + r] + first[r] : first[r]) + second[r];
  }
}

// Whether the gradients' one-hot rows have one array instead of two: where LDS holds no more.
template <typename T, int D, int ST>
constexpr bool one_hot() {
  return 4 * kTile * Tile<T, D>::kRow + 2 * HotTile<ST>::kBytes + kMostValues * 4 + 2048 > 160 * 1024;
}

int check_buckets(const ctmr_masked_attention_desc* d, const ctmr_buckets_desc* b);
Bias make_bias(const ctmr_masked_attention_desc* d, const ctmr_buckets_desc* b, const void* plan, const void* table);
int bias_steps(const ctmr_buckets_desc* b);  // contraction steps that the kernels have

// The gradients' kernels for heads of T.
template <typename T>
int run_biased_gradients(const Args& a, const Bias& bias, int steps, int qparts, int kparts, hipStream_t st);
template <>
int run_biased_gradients<float>(const Args&, const Bias&, int, int, int, hipStream_t);
template <>
int run_biased_gradients<__bf16>(const Args&, const Bias&, int, int, int, hipStream_t);
template <>
int run_biased_gradients<_Float16>(const Args&, const Bias&, int, int, int, hipStream_t);

// Bytes of the values in LDS, the kernels' dynamic part.
template <typename T, int D>
inline unsigned bias_bytes(const Bias& b) { return kSingle<T, D> ? 4096u : 4u * b.values; }
template <typename T, int D>
inline unsigned bias_bytes(const BiasOf<0>&) { return 0u; }

}  // namespace attn
}  // namespace ctmr
