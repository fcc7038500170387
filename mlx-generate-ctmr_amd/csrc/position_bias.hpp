// A learned bias of attention scores by the distance of a row and a key on each of
// up to four axes, in matrix products.
//
//   bias_ij = sum_a table[row_a(x_a(j) - x_a(i))][h]
// where x_a is a token's place on axis a, 0 .. extent_a - 1, and row_a the table's row
// for a distance (its bucket).  For a query row i that is a function of the key's place
// on each axis, so with a column c = (a, x) for each place of each axis
//   bias_ij = sum_c r_i[c] o_j[c],  r_i[a, x] = table[row_a(x - x_a(i))][h],  o_j[a, x] = (x_a(j) == x)
// and likewise with the sides exchanged, r'_j[a, x] = table[row_a(x_a(j) - x)][h].  The
// table's gradient is that of r_i, which is one product more over the scores' gradients,
//   dr_i[c] = sum_j ds_ij o_j[c],
// added up over the distances of each row of the table.
//
// The one-hot rows o are exact in bf16 and the same for all heads: they stream through
// LDS beside the keys (or the query rows).  r has kParts bf16 parts, whose products with
// o are exact, so the bias is r to 2^-17 (16-bit heads; their weights are rounded by
// 2^-9 or 2^-12) or to all of fp32's bits (fp32 heads); ds likewise.  A wave keeps r as
// the B operand.
#pragma once

#include "masked_attention.hpp"

namespace ctmr {
namespace attn {

constexpr int kColumns = 128;   // at most, over all axes
constexpr int kNumbers = 512;   // of distances: two for a column, and room past them for columns that no place has
constexpr int kDistances = 256;  // numbers that a distance may have

// A plan of places (ctmr_buckets), and the table.
struct Bias {
  const int* rows;           // (kNumbers) the table's row of a distance's number, -1 for none
  const int* query_columns;  // (kColumns) axis << 16 | the number of column c's distance from place 0
  const int* key_columns;    // likewise to place 0
  const unsigned *query_places, *key_places;  // (items, rows) a byte for each axis
  const __bf16 *query_hot, *key_hot;          // (items, rows, 16 ST) o
  int64_t query_item, key_item;               // rows from item to item (0: all have the same)
  const void* table;         // (table_rows, hq)
  int elem, table_rows, axes;
  int extents[4], first_column[4], first_number[4];  // of each axis
  bool fine;    // forward, 16-bit heads: weights in two parts (see fine_weights)
  float* part;  // the gradient: (n, hq, slots, kDistances) sums over a block's rows, or null
  int slots;
};

// ST: contraction steps of 16 columns, 3, 4, 6 or 8; 0: no bias.
template <int ST>
struct BiasOf : Bias {
  static constexpr int kSteps = ST, kBlocks = (ST + 1) / 2;  // 32-column blocks
  static constexpr int kRow = 16 * ST;                       // columns of a row of o in memory
  static constexpr int kWidth = ST <= 4 ? 64 : 128;          // and of a tile in LDS, zeros past them
};
template <>
struct BiasOf<0> {
  static constexpr int kSteps = 1, kBlocks = 1, kRow = 32, kWidth = 32;  // of arrays that nothing uses
};

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 2;

// A lane's r of one row, in parts.
template <typename T, int ST>
struct BiasRow {
  Frag<__bf16> part[BiasOf<ST>::kSteps][kParts<T>];
};

// The table's value for a distance's number, in units of 1 / `unit`.  What is below -2^100 hides a pair: the score that it
// makes is below kNone in log2 units (the host keeps c from 2^-20), and zero times it is zero.
__device__ __forceinline__ float bias_value(const Bias& b, int number, int h, int hq, float unit) {
  const int row = b.rows[number];
  if (row < 0) return 0.f;
  const float v = load_param(b.table, b.elem, (int64_t)row * hq + h);
  return v < -0x1p100f ? -0x1p127f : v * unit;
}

// r of a row at `places` for head h.  KEYS: of a key (r').
template <typename T, int ST, bool KEYS>
__device__ __forceinline__ void bias_row(const Bias& b, BiasRow<T, ST>& out, unsigned places, int h, int hq, float unit,
                                         int lane) {
  const int* columns = KEYS ? b.key_columns : b.query_columns;
#pragma unroll
  for (int n = 0; n < ST; ++n)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = columns[16 * n + 8 * (lane >> 5) + e];
      const int place = (places >> (8 * (c >> 16))) & 255, number = (c & 0xffff) + (KEYS ? place : -place);
      float v = bias_value(b, number, h, hq, unit);
#pragma unroll
      for (int p = 0; p < kParts<T>; ++p) {
        const __bf16 part = (__bf16)v;
        out.part[n][p][e] = part;
        v -= (float)part;
      }
    }
}

// Adds the bias of 32 rows of one-hot values in LDS to raw scores.
template <typename T, int ST>
__device__ __forceinline__ void add_bias(f16v& s, const BiasRow<T, ST>& r, const char* hot, int row, int lane) {
#pragma unroll
  for (int n = 0; n < ST; ++n) {
    const Frag<__bf16> o = Tile<__bf16, BiasOf<ST>::kWidth>::along(hot, row, n, lane);
#pragma unroll
    for (int p = 0; p < kParts<T>; ++p) s = mma<__bf16>(o, r.part[n][p], s);
  }
}

// Whether the one-hot rows of a bias have one array instead of two: where LDS holds no more.
template <typename T, int D, int ST>
constexpr bool one_hot() {
  return 4 * kTile * Tile<T, D>::kRow + 4 * kTile * BiasOf<ST>::kWidth + 2048 > 160 * 1024;
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

}  // namespace attn
}  // namespace ctmr
