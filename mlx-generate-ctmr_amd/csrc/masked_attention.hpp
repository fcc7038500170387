// What the forward and backward kernels of the masked attention share: MFMA
// fragments of fp32, bf16 and fp16 operands, tiles of rows in LDS, scores and
// masks.
//
// Scores of query row i and key j of one head, in log2 units:
//   s = scale q_i . k_j;  s = cap tanh(s / cap) with a cap;  s -= slope |p_i - j|
//   with slopes, p_i = i + lk - lq;  s2 = s log2(e)
// Key j is visible to row i if j < limit_i = min(lk, max(p_i + 1, prefix)) (lk without
// a prefix) and, with documents, id_i = id_j >= 0.
//
// Every product runs on 32x32 MFMA tiles in one orientation: the matrix that
// streams through LDS gives the rows (A), the one that a wave keeps in registers
// the columns (B), so that a lane holds 16 of a column's 32 results:
//   lane l, register r -> row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32.
// A contraction step takes 16 places, eight for each half of the wave.  Which
// eight is free as long as A and B agree: operands read along their rows take 8
// (l / 32) .. + 7; results that are operands of the next product take the rows the
// lane holds, 4 (l / 32) + {0..3, 8..11}, so they never cross lanes, and the other
// operand is read from LDS down its columns in that order.
#pragma once

#include "elements.hpp"

#include <type_traits>

namespace ctmr {
namespace attn {

constexpr int kTile = 64;      // rows of a streamed tile
constexpr float kNone = -1e30f;  // running maximum before any visible key, in log2 units
constexpr float kLog2e = 1.44269504f;

typedef Vec<float, 16> f16v;

template <typename T>
using Frag = Vec<T, 8>;

template <typename T>
__device__ __forceinline__ f16v mma(const Frag<T>& a, const Frag<T>& b, f16v c) {
  if constexpr (std::is_same_v<T, __bf16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  } else if constexpr (std::is_same_v<T, _Float16>) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
}

// Eight results of a lane (registers 8 step .. + 7) as an operand, rounded to T.
template <typename T>
__device__ __forceinline__ Frag<T> result_frag(const f16v& s, int step) {
  Vec<float, 8> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = s[8 * step + e];
  return __builtin_convertvector(v, Frag<T>);
}

// Values and bytes between rows of a tile in LDS.  ALONG: read along its rows only,
// 16 bytes a lane from 32 rows (16 bytes of padding spread them over the banks);
// DOWN: down its columns only, four rows of 64 bytes at a time (rows 64 bytes
// apart modulo 256); BOTH: 32 bytes of padding, a conflict of two either way.
enum Reads { ALONG, DOWN, BOTH };
template <typename T, int D>
constexpr int tile_stride(Reads r) {
  if (sizeof(T) == 4) return D + 4;
  if (r == ALONG) return D + 8;
  if (r == BOTH) return D + 16;
  return D == 32 ? 32 : D + 32;
}

// A operand of 32 rows from `row`, contraction over the values 16 step .. + 15 of a row.
template <typename T>
__device__ __forceinline__ Frag<T> frag_along(const T* tile, int stride, int row, int step, int lane) {
  const T* p = tile + (row + (lane & 31)) * stride + 16 * step + 8 * (lane >> 5);
  return *reinterpret_cast<const Frag<T>*>(p);
}

// A operand whose rows are the values 32 block .. + 31, contraction over the tile's rows `row` .. + 15 in the
// results' order.
template <typename T>
__device__ __forceinline__ Frag<T> frag_down(const T* tile, int stride, int row, int block, int lane) {
  const int half = lane >> 5;
  if constexpr (sizeof(T) == 4) {
    const T* p = tile + (row + 4 * half) * stride + 32 * block + (lane & 31);
    Frag<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = p[(e + (e & 4)) * stride];
    return f;
  } else {
    // A transposing read: of 16 lanes, lane m gives the address of four values of row m / 4 and gets column m
    // of the four rows.
    typedef Vec<short, 4> s4;
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const T* p = tile + (row + 4 * half + ((lane & 15) >> 2)) * stride + 32 * block + 16 * ((lane >> 4) & 1) +
                 4 * (lane & 3);
    const s4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
    const s4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * stride));
    return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// B operand of a wave's 32 rows straight from memory: this lane's row, zeros where `valid` is false or past d values.
template <typename T>
__device__ __forceinline__ Frag<T> frag_global(const T* row, int step, int d, int lane, bool valid) {
  const int at = 16 * step + 8 * (lane >> 5);
  Frag<T> f = Frag<T>(0);
  if (valid && at < d) f = *reinterpret_cast<const Frag<T>*>(row + at);
  return f;
}

// --------------------------------------------------------------------------
// streaming a tile: memory -> registers -> LDS, 16 bytes a thread and piece
// --------------------------------------------------------------------------
template <typename T, int D, int ROWS, int THREADS>
struct Stream {
  static constexpr int kPer = 16 / (int)sizeof(T);            // values of a piece
  static constexpr int kPieces = ROWS * D / kPer / THREADS;   // of a thread
  static_assert(ROWS * D % (kPer * THREADS) == 0, "whole pieces");
  u4 piece[kPieces];

  static __device__ __forceinline__ int row_of(int i, int t) { return (i * THREADS + t) / (D / kPer); }
  static __device__ __forceinline__ int col_of(int i, int t) { return (i * THREADS + t) % (D / kPer) * kPer; }

  // Rows first .. first + ROWS - 1 of `rows` (strides in values, d values each); zeros past either end.  The
  // buffer's range ends with the last row; a column past d has an offset past every range.  The host keeps
  // kTile * stride bytes below 2^31.
  __device__ __forceinline__ void fetch(const T* base, int64_t stride, int first, int rows, int d, int t) {
    const int left = min(rows - first, ROWS);
    const int bytes = left > 0 ? (int)(((int64_t)(left - 1) * stride + d) * (int)sizeof(T)) : 0;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)first * stride), (short)0, bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i, t), col = col_of(i, t);
      const int off = col < d ? (int)((row * stride + col) * (int)sizeof(T)) : 0x7ffffff0;
      piece[i] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    }
  }

  // CLEAN: values that are not finite become zeros and their rows' bits are set in odd[ROWS / 32].
  template <bool CLEAN>
  __device__ __forceinline__ void store(T* tile, int stride, unsigned* odd, int t) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i, t);
      if constexpr (CLEAN) {
        bool found = false;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          unsigned u = piece[i][w];
          if constexpr (sizeof(T) == 4) {
            if ((u & 0x7f800000u) == 0x7f800000u) u = 0u;
          } else {
            constexpr unsigned kExp = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u;
            if ((u & kExp) == kExp) u &= 0xffff0000u;
            if ((u & (kExp << 16)) == (kExp << 16)) u &= 0x0000ffffu;
          }
          found |= u != piece[i][w];
          piece[i][w] = u;
        }
        if (found) atomicOr(&odd[row >> 5], 1u << (row & 31));
      }
      *reinterpret_cast<u4*>(tile + row * stride + col_of(i, t)) = piece[i];
    }
  }
};

// --------------------------------------------------------------------------
// arguments, masks and scores
// --------------------------------------------------------------------------
struct DocTile {     // of kTile rows: ids of all its rows, and of those that are no padding
  int least, most, least_id, unused;
};
constexpr int kGrain = 32;  // rows of a hull: a wave's

struct Side {        // documents of the query or key rows
  const int* ids;    // (n, rows rounded up to kTile), -1 past the end
  const DocTile* tiles;
  const int4* hull;  // of kGrain rows, tiles of the other side: [x, y) may hold a match, all pairs with [z, w) are one
  int stride, count, grains;  // ids, tiles and hulls of a batch item
};

struct Args {
  const void *q, *k, *v;
  void* out;
  void* rest;             // what rounding took from out, as out lies, or null
  float* lse;             // (n, hq, lq) log2 of a row's sum, +inf for an empty row
  float* part;            // split keys: (splits, n, hq, lq, D) sums, then (.., 2) maximum and total
  const void* dout;
  void *dq, *dk, *dv;
  float* delta;           // (n, hq, lq) sum_d dout out
  const float* slopes;    // (hq)
  const int* prefixes;    // (n), or null with `prefix`
  Side qdoc, kdoc;        // ids null: no documents
  int64_t qb, qh, ql, kb, kh, kl, vb, vh, vl, ob, oh, ol, gb, gh, gl;  // strides; g: dout
  int64_t dqb, dqh, dql, dkb, dkh, dkl, dvb, dvh, dvl;
  int n, lq, lk, hq, hk, group, d;
  int prefixed, prefix, splits;
  float scale, cap;
};

__device__ __forceinline__ int prefix_of(const Args& a, int b) { return a.prefixes ? a.prefixes[b] : a.prefix; }

// First key that row i can no longer see, documents aside.
__device__ __forceinline__ int limit_of(const Args& a, int i, int prefix) {
  return a.prefixed ? min(a.lk, max(i + a.lk - a.lq + 1, prefix)) : a.lk;
}

// What a row compares key ids with: its own id, -2 where it is padding.
__device__ __forceinline__ int row_id(const Args& a, int b, int i) {
  const int id = a.qdoc.ids[(int64_t)b * a.qdoc.stride + i];
  return id < 0 ? -2 : id;
}

// tanh to about 2e-7 absolute: enough for 16-bit operands, whose scores it moves by under 2^-17 at a cap of 50.
template <typename T>
__device__ __forceinline__ float tanh_of(float x) {
  if constexpr (sizeof(T) == 4) {
    return tanhf(x);
  } else {
    const float e = __builtin_amdgcn_exp2f(2.0f * kLog2e * x);
    return fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  }
}

__device__ __forceinline__ float half_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// Item and tile of a workgroup: blocks go round the eight XCDs, each of which has
// its own L2, so all tiles of a (batch item, head) that stream the same rows go to
// one of them where the items divide by eight.
__device__ __forceinline__ void place(int id, int items, int tiles, int& item, int& tile) {
  if (items % 8 == 0) {
    const int rest = id >> 3;
    item = rest / tiles * 8 + (id & 7);
    tile = rest % tiles;
  } else {
    item = id / tiles;
    tile = id % tiles;
  }
}

// Tiles that kGrain rows of one side meet: [x, y) may hold visible pairs, in [z, w) every pair is visible.
__device__ __forceinline__ int4 meet(const Side& s, int b, int grain, int4 r) {
  if (s.ids) {
    const int4 hull = s.hull[(int64_t)b * s.grains + grain];
    r = {max(r.x, hull.x), min(r.y, hull.y), max(r.z, hull.z), min(r.w, hull.w)};
  }
  r.y = max(r.y, 0);
  r.x = min(r.x, r.y);
  return r;
}

// Key tiles of the rows i .. i + kGrain - 1 of item b, those past lq aside.
__device__ __forceinline__ int4 key_tiles(const Args& a, int b, int i, int prefix) {
  const int last = limit_of(a, min(i + kGrain, a.lq) - 1, prefix), first = limit_of(a, i, prefix);
  return meet(a.qdoc, b, i / kGrain, int4{0, (max(last, 0) + kTile - 1) / kTile, 0, max(first, 0) / kTile});
}

// Query tiles of the keys j .. j + kGrain - 1: from the first row whose limit passes j; every key is seen from the
// row whose limit passes the last one.
__device__ __forceinline__ int4 query_tiles(const Args& a, int b, int j, int prefix) {
  const int end = min(j + kGrain, a.lk) - 1, off = a.lk - a.lq, tiles = (a.lq + kTile - 1) / kTile;
  const int first = a.prefixed && prefix <= j ? max(0, j - off) / kTile : 0;
  const int whole = a.prefixed && prefix <= end ? (max(0, end - off) + kTile - 1) / kTile : 0;
  return meet(a.kdoc, b, j / kGrain, int4{first, tiles, whole, tiles});
}

// A workgroup's tiles from its waves' (those with rows): any may hold a pair, all are whole.
struct Meeting {
  int4 mine, all;
  __device__ __forceinline__ bool partial(int tile) const { return tile < all.z || tile >= all.w; }
  __device__ __forceinline__ bool skips(int tile) const { return tile < mine.x || tile >= mine.y; }
  __device__ __forceinline__ bool masked(int tile) const { return tile < mine.z || tile >= mine.w; }
};
template <int WAVES, typename F>
__device__ __forceinline__ Meeting meeting(int wave, int row0, int rows, F tiles_of) {
  Meeting m;
  m.mine = int4{0, 0, 0, 0};
  m.all = int4{0x7fffffff, 0, 0, 0x7fffffff};
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int row = row0 + kGrain * w;
    if (row >= rows) break;
    const int4 r = tiles_of(row);
    if (r.x < r.y) {
      m.all.x = min(m.all.x, r.x);
      m.all.y = max(m.all.y, r.y);
    }
    m.all.z = max(m.all.z, r.z);
    m.all.w = min(m.all.w, r.w);
    if (w == wave) m.mine = r;
  }
  m.all.x = min(m.all.x, m.all.y);
  return m;
}

int check_desc(const ctmr_masked_attention_desc* d);
int padded(int head_dim);
Args make_args(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const float* slopes,
               const int32_t* prefixes, const void* plan);

}  // namespace attn
}  // namespace ctmr
