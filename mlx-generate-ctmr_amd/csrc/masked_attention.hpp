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

// A value that is the same for the wave, in a scalar register of its own: the kernel's arguments come in blocks of
// up to 16 registers, and a loop that needs one value of each spills them.
template <typename V>
__device__ __forceinline__ V apart(V v) {
  asm("" : "+s"(v));
  return v;
}

// The lane, unknown to the compiler: the permuted addresses of a tile's reads are then computed where they are used
// (one exclusive or each) instead of held in registers over the loop, for kernels that have none to spare.
template <bool HIDE>
__device__ __forceinline__ int fresh(int lane) {
  if constexpr (HIDE) asm volatile("" : "+v"(lane));
  return lane;
}

// A tile of D-value rows in LDS, in pieces of 16 bytes.  The pieces of a row are
// permuted by the row (an exclusive or) so that no read meets a bank twice in the 256
// bytes that LDS moves a cycle, without padding: along, sixteen lanes read one piece of
// sixteen rows; down, 32 lanes read 64 bytes of four rows, or in fp32 64 lanes read 128
// bytes of rows r and r + 4 (rows of 128 bytes keep a conflict of two there).
template <typename T, int D>
struct Tile {
  static constexpr int kRow = D * (int)sizeof(T);  // bytes
  static constexpr int kPieces = kRow / 16;        // 4, 8, 16 or 32

  static __device__ __forceinline__ int mix(int r) {
    if constexpr (kPieces == 4) return (r >> 2) & 3;
    if constexpr (kPieces == 8) return ((r << 1) & 4) | ((r >> 2) & 3);
    if constexpr (sizeof(T) == 4) return ((r << 1) & 8) | ((r << 1) & 6) | ((r >> 3) & 1);
    return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int row, int piece) { return row * kRow + ((piece ^ mix(row)) << 4); }

  // A operand of the 32 rows from `row` (a multiple of 16), contraction over the values 16 step .. + 15 of a row.
  static __device__ __forceinline__ Frag<T> along(const char* tile, int row, int step, int lane) {
    const char* p = tile + row * kRow;
    const int r = lane & 31, half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const Frag<T>*>(p + at(r, 2 * step + half));
    } else {
      const f4 u = *reinterpret_cast<const f4*>(p + at(r, 4 * step + 2 * half));
      const f4 w = *reinterpret_cast<const f4*>(p + at(r, 4 * step + 2 * half + 1));
      return __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  // A operand whose rows are the values 32 block .. + 31, contraction over the tile's rows `row` .. + 15 (a
  // multiple of 16) in the results' order.
  static __device__ __forceinline__ Frag<T> down(const char* tile, int row, int block, int lane) {
    const char* p = tile + row * kRow;
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 4) {
      Frag<T> f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        f[e] = *reinterpret_cast<const T*>(p + at(4 * half + e + (e & 4), 8 * block + ((lane & 31) >> 2)) +
                                           4 * (lane & 3));
      return f;
    } else {
      // A transposing read: of 16 lanes, lane m gives the address of four values of row m / 4 and gets column m
      // of the four rows.
      typedef Vec<short, 4> s4;
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const int r = 4 * half + ((lane & 15) >> 2), piece = 4 * block + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      const s4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + at(r, piece) + 8 * (lane & 1)));
      const s4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + at(r + 8, piece) + 8 * (lane & 1)));
      return __builtin_bit_cast(Frag<T>, __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

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
// The rows of one head from some row on, walked ROWS at a time; the same for all threads.  The host keeps kTile *
// stride bytes below 2^30.
template <typename T, int ROWS>
struct Rows {
  const char* base;
  int64_t step;     // bytes of ROWS rows
  int left;       // rows
  int row, last;  // bytes of a row's stride and of its values

  __device__ __forceinline__ void begin(const T* rows, int64_t stride, int first, int count, int d) {
    row = apart((int)(stride * (int)sizeof(T)));
    last = apart(d * (int)sizeof(T));
    step = (int64_t)ROWS * row;
    base = reinterpret_cast<const char*>(rows + (int64_t)first * stride);
    left = count - first;
  }
  __device__ __forceinline__ void next() {
    base += step;
    left -= ROWS;
  }
  // Loads past the last row give zeros.
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer() const {
    const int bytes = max((min(left, ROWS) - 1) * row + last, 0);
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
  }
};

// Every thread's loads into LDS are there, and the reads before it are done.
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

// A wave's 64 floats from place `first` of `count` straight into LDS, zeros past the end.  Complete after arrive().
__device__ __forceinline__ void load_floats(float* to, const float* from, int first, int count, int lane) {
  typedef __attribute__((address_space(3))) void lds_void;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(from + first), (short)0, max(min(count - first, 64), 0) * 4, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)to, 4, lane * 4, 0, 0, 0);
}

template <typename T, int D, int ROWS, int THREADS>
struct Stream {
  typedef Tile<T, D> Lds;
  static constexpr int kPieces = ROWS * Lds::kPieces / THREADS;  // of a thread
  static_assert(ROWS * Lds::kPieces % THREADS == 0, "whole pieces");
  u4 piece[kPieces];

  static __device__ __forceinline__ int row_of(int i, int t) { return (i * THREADS + t) / Lds::kPieces; }
  static __device__ __forceinline__ int piece_of(int t) { return t % Lds::kPieces; }  // THREADS is a multiple

  // Whether 16 bytes hold finite values only; those that are not become zeros.
  static __device__ __forceinline__ bool finite(u4& v) {
    bool all = true;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      unsigned u = v[w];
      if constexpr (sizeof(T) == 4) {
        if ((u & 0x7f800000u) == 0x7f800000u) u = 0u;
      } else {
        constexpr unsigned kExp = std::is_same_v<T, __bf16> ? 0x7f80u : 0x7c00u;
        if ((u & kExp) == kExp) u &= 0xffff0000u;
        if ((u & (kExp << 16)) == (kExp << 16)) u &= 0x0000ffffu;
      }
      all &= u == v[w];
      v[w] = u;
    }
    return all;
  }

  // Columns past the head's values have an offset past every range, 2^30 + 2^29 and more.
  __device__ __forceinline__ void fetch(const Rows<T, ROWS>& rows, int t) {
    const __amdgpu_buffer_rsrc_t r = rows.buffer();
    unsigned off = row_of(0, t) * rows.row + piece_of(t) * 16;
    off = piece_of(t) * 16 < rows.last ? off : 0x60000000u;
#pragma unroll
    for (int i = 0; i < kPieces; ++i)
      piece[i] = __builtin_amdgcn_raw_buffer_load_b128(r, (int)(off + i * (THREADS / Lds::kPieces) * rows.row), 0, 0);
  }

  // Straight into LDS: a wave's lanes write 16 bytes each side by side, so the permutation is done on the memory's
  // side.  Complete after arrive().  The two arrays of a kernel are separate, so that the compiler knows that reads of
  // one do not wait for what is on its way into the other.
  static __device__ __forceinline__ void load(char* tile, const Rows<T, ROWS>& rows, int t) {
    typedef __attribute__((address_space(3))) void lds_void;
    const __amdgpu_buffer_rsrc_t r = rows.buffer();
    char* wave = tile + __builtin_amdgcn_readfirstlane(t & ~63) * 16;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i, t), piece = piece_of(t) ^ Lds::mix(row);
      const unsigned off = piece * 16 < rows.last ? row * rows.row + piece * 16 : 0x60000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(wave + i * THREADS * 16), 16, (int)off, 0, 0, 0);
    }
  }

  // Of a tile in LDS: values that are not finite become zeros and their rows' bits are set in odd[ROWS / 32].
  static __device__ __forceinline__ void clean(char* tile, unsigned* odd, int t) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      u4* at = reinterpret_cast<u4*>(tile + (i * THREADS + t) * 16);
      u4 v = *at;
      if (finite(v)) continue;
      *at = v;
      const int row = row_of(i, t);
      atomicOr(&odd[row >> 5], 1u << (row & 31));
    }
  }

  // CLEAN: values that are not finite become zeros and their rows' bits are set in odd[ROWS / 32].
  template <bool CLEAN>
  __device__ __forceinline__ void store(char* tile, unsigned* odd, int t) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int row = row_of(i, t);
      if constexpr (CLEAN) {
        if (!finite(piece[i])) atomicOr(&odd[row >> 5], 1u << (row & 31));
      }
      *reinterpret_cast<u4*>(tile + Lds::at(row, piece_of(t))) = piece[i];
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
constexpr int kBlockRows = 128;  // rows of a workgroup of four waves

struct Side {        // documents of the query or key rows
  const int* ids;    // (n, rows rounded up to kTile), -1 past the end
  const DocTile* tiles;
  // Three for kGrain rows: tiles of the other side, [x, y) that may hold a match of the first row's document and
  // [z, w) that hold nothing else; the same of the other rows' documents ([z, w) empty if they are of several, or
  // padding is among them); the least and the largest id of these (-1: padding), x > y if there are none.
  const int4* hull;
  const int* mixed;  // whether kBlockRows rows are of more than one document
  int stride, count, grains;  // ids, tiles and hulls of a batch item
};

struct Args {
  const void *q, *k, *v;
  void* out;
  void* rest;             // what rounding took from out, as out lies, or null
  float* lse;             // (n, hq, lq) log2 of a row's sum (with a shifted cap: of the scores less cap), +inf for an
                          // empty row
  float* part;            // split keys: (splits, n, hq, lq, D) sums, then (.., 2) maximum and total
  const void* dout;
  void *dq, *dk, *dv;
  float* delta;           // (n, hq, lq) -sum_d dout out
  const float* slopes;    // (hq)
  const int* prefixes;    // (n), or null with `prefix`
  Side qdoc, kdoc;        // ids null: no documents
  int64_t qb, qh, ql, kb, kh, kl, vb, vh, vl, ob, oh, ol, gb, gh, gl;  // strides; g: dout
  int64_t dqb, dqh, dql, dkb, dkh, dkl, dvb, dvh, dvl;
  int n, lq, lk, hq, hk, group, d;
  int prefixed, prefix, splits;
  float scale, cap;
};

// What scores of one head are made of, apart.
struct Scoring {
  float scale, cap, slope;
  bool sloped, prefixed;
};
__device__ __forceinline__ Scoring scoring_of(const Args& a, int h) {
  return {apart(a.scale), apart(a.cap), a.slopes ? a.slopes[h] : 0.f, a.slopes != nullptr, a.prefixed != 0};
}

__device__ __forceinline__ int prefix_of(const Args& a, int b) { return a.prefixes ? a.prefixes[b] : a.prefix; }

// First key that row i can no longer see, documents aside.
__device__ __forceinline__ int limit_of(const Args& a, int i, int prefix) {
  return a.prefixed ? min(a.lk, max(i + a.lk - a.lq + 1, prefix)) : a.lk;
}

// Document of a query row; negative is padding, which compares as -2 with ids that are -1 at least.
__device__ __forceinline__ int id_of(const Args& a, int b, int i) {
  return a.qdoc.ids[(int64_t)b * a.qdoc.stride + i];
}

// Forms of the cap, t = tanh(x per) of a raw product x, each in kernels of its own (a choice at run time takes a wave a
// SIMD from the forward kernels' registers).  Exact: t itself, in fp32 and for caps past kShiftedMost.
// Shifted, 16-bit operands: (t - 1) / 2 = -1 / (1 + e^(2 x per)), one operation less; the softmax does not see the shift,
// and lse has it too.  The hardware's exponential and reciprocal are exact to about 1e-7, which near -1/2, where small
// scores lie, is an error of the score of 1e-7 caps whatever the score: 2e-5 at most, where fp16 rounds weights by 2e-4.
// Forward, 2 x 16 heads of 4096 rows of 64, bf16: no cap 167 us, shifted 223, exact 334; gradients 497, 671, 858.
enum Cap { kNoCap, kShiftedCap, kExactCap };
constexpr float kShiftedMost = 256.0f;
template <typename T>
inline bool shifted_cap(float cap) {
  return sizeof(T) == 2 && cap <= kShiftedMost;
}
// Of t in what is returned.
template <Cap CAP>
constexpr float kCapUnits = CAP == kShiftedCap ? 2.0f : 1.0f;
template <Cap CAP>
__device__ __forceinline__ void cap_scores(f16v& s, float per) {
  if constexpr (CAP == kExactCap) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = tanhf(s[r] * per);
  } else {
    // Operation by operation: chained score by score they wait for each other (2 x 16 heads of 4096 rows of 128 behind
    // a prefix: 273 us, 266 so).
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] * (per * (2.0f * kLog2e)));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = -1.0f - s[r];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_rcpf(s[r]);
  }
}
// 1 - t^2 of it, in units of kCapSlope.
template <Cap CAP>
constexpr float kCapSlope = CAP == kShiftedCap ? -4.0f : 1.0f;
template <Cap CAP>
__device__ __forceinline__ float cap_slope(float s) {
  return CAP == kExactCap ? fmaf(-s, s, 1.0f) : fmaf(s, s, s);
}

__device__ __forceinline__ float half_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// Item, tile and part of a workgroup: blocks go round the eight XCDs, each of which
// has its own L2, so all tiles of a (batch item, head) that stream the same rows go
// to one of them where the items divide by eight.
//
// With documents two workgroups share a block of rows (parts 2): part 0 takes the
// rows of the first row's document, part 1 the others.  A block that two long
// documents meet in would else walk both, twice as long as any other: of 6144
// tokens in documents of 2048, 1573, 2048 and 400, 16 heads of 32, that one block a
// head made 2.6 times the time with the borders on block borders; so 1.07 times.
__device__ __forceinline__ void place(int id, int items, int tiles, int parts, int& item, int& tile, int& part) {
  const bool spread = items % 8 == 0;
  int rest = spread ? id >> 3 : id;
  part = 0;
  if (parts == 2) {  // the second parts first: most have no rows and leave at once
    const int each = spread ? items / 8 * tiles : items * tiles;
    part = rest < each ? 1 : 0;
    rest -= part ? 0 : each;
  }
  item = spread ? rest / tiles * 8 + (id & 7) : rest / tiles;
  tile = rest % tiles;
}

// The rows of a workgroup's part: those whose id is (part 0) or is not (part 1) `first_id`.
struct Part {
  int part, first_id;
  __device__ __forceinline__ bool has(int id) const { return (id == first_id) == (part == 0); }
};

// Whether a block of rows has a second part.
__device__ __forceinline__ bool is_mixed(const Side& s, int b, int block) {
  return s.mixed[(int64_t)b * ((s.grains + 3) / 4) + block] != 0;
}

// Tiles that kGrain rows of one side meet: [x, y) may hold visible pairs, in [z, w) every pair is visible.  With
// documents and a part only the part's rows count.
__device__ __forceinline__ int4 meet(const Side& s, int b, int grain, int4 r, const Part* part) {
  if (s.ids) {
    const int4* hull = s.hull + 3 * ((int64_t)b * s.grains + grain);
    const int4 ids = hull[2];
    const bool first = !part || part->has(s.ids[(int64_t)b * s.stride + grain * kGrain]);
    const bool others = ids.x <= ids.y &&
                        (!part || part->part == 1 || (ids.x <= part->first_id && part->first_id <= ids.y));
    int4 u = {0x7fffffff, 0, 0x7fffffff, 0};
    if (first) u = hull[0];
    if (others) {
      const int4 o = hull[1];
      u = {min(u.x, o.x), max(u.y, o.y), first ? 0x7fffffff : o.z, first ? 0 : o.w};
    }
    r = {max(r.x, u.x), min(r.y, u.y), max(r.z, u.z), min(r.w, u.w)};
  }
  r.y = max(r.y, 0);
  r.x = min(r.x, r.y);
  return r;
}

// Key tiles of the rows i .. i + kGrain - 1 of item b, those past lq aside.
__device__ __forceinline__ int4 key_tiles(const Args& a, int b, int i, int prefix, const Part* part) {
  const int last = limit_of(a, min(i + kGrain, a.lq) - 1, prefix), first = limit_of(a, i, prefix);
  return meet(a.qdoc, b, i / kGrain, int4{0, (max(last, 0) + kTile - 1) / kTile, 0, max(first, 0) / kTile}, part);
}

// Query tiles of the keys j .. j + kGrain - 1: from the first row whose limit passes j; every key is seen from the
// row whose limit passes the last one, up to the last whole tile.
__device__ __forceinline__ int4 query_tiles(const Args& a, int b, int j, int prefix, const Part* part) {
  const int end = min(j + kGrain, a.lk) - 1, off = a.lk - a.lq, tiles = (a.lq + kTile - 1) / kTile;
  const int first = a.prefixed && prefix <= j ? max(0, j - off) / kTile : 0;
  const int whole = a.prefixed && prefix <= end ? (max(0, end - off) + kTile - 1) / kTile : 0;
  return meet(a.kdoc, b, j / kGrain, int4{first, tiles, whole, a.lq / kTile}, part);
}

// A workgroup's tiles from its waves' (those that meet any): any wave may hold a pair, all waves' are whole.
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
      m.all.z = max(m.all.z, r.z);
      m.all.w = min(m.all.w, r.w);
    }
    if (w == wave) m.mine = r;
  }
  m.all.x = min(m.all.x, m.all.y);
  return m;
}

int check_desc(const ctmr_masked_attention_desc* d);
int check_strides(const ctmr_masked_attention_desc* d, const int64_t* strides, int rows);
int64_t row_stride(const int64_t* strides, int rows, int head_dim);  // of one row: any that does not overlap
int padded(int head_dim);
Args make_args(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const float* slopes,
               const int32_t* prefixes, const void* plan);

}  // namespace attn
}  // namespace ctmr
