// Attention with grouped heads, a tanh cap, a distance bias, documents and a
// prefix: forward, for fp32, bf16 and fp16 heads of up to 128 values.
//
//   out_i = sum_j p_ij v_j,  p_ij = 2^(s2_ij - lse_i),  lse_i = log2 sum_j 2^s2_ij
// over the keys visible to row i (masked_attention.hpp); a row that sees none is zero.
//
// One pass over the keys: S^T = K Q^T per 64-key tile, the running maximum m and
// sum l of each row, O^T += V^T P^T.  m follows a row's maximum only when it is
// passed by 8 (in log2 units), so the outputs are rarely rescaled and P stays below
// 2^8; m, l and O are fp32.  P is rounded to the operands' type for the second
// product, half a step of that type on each weight, as the output's own rounding: 16-bit
// outputs are 1.4 times as far from 64 bits as rounding alone leaves them (bf16 2.3e-3
// for 1.7e-3, fp16 2.9e-4 for 2.1e-4).
//
// Masked places have no effect whatever they hold: masked scores are replaced, and
// in tiles with masked places the values of V that are not finite are zeroed on
// their way into LDS (0 * NaN) and added to the rows that do see them afterwards.
//
// Bound by the softmax's vector operations (five a score: fma, exp, a sum, half a
// maximum, half a conversion) with heads of 32 and 64, by them and the matrix products
// in turn with 128: bf16, 2 x 16 heads of 4096 rows, every key: heads of 32 116 us
// (592 TFLOP/s), of 64 163 (843), of 128 270 (1018); fp32, 2 x 8 heads of 2048 rows of
// 32: 84 us, 102 TFLOP/s of the products alone, which run at 153 at best.
#pragma once

#include "position_bias.hpp"

#include <algorithm>
#include <cmath>

namespace ctmr {
namespace attn {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRows = kBlockRows;  // query rows of a workgroup of the tiled form
static_assert(kRows == 32 * kWaves && kRows == 4 * kGrain, "32 rows a wave");
constexpr float kLazy = 8.0f;
// fp16 weights are raised by 2^6 (both in O and l): below 2^8 * 2^6 they stay in range, and weights down to
// 2^-20 of the reference keep all their bits.
template <typename T>
constexpr float kLift = std::is_same_v<T, _Float16> ? 6.0f : 0.0f;

// What this lane's row may see: keys below limit whose id is id.
struct RowMask {
  int limit, id;
};

// Raw products of NB 32-key blocks -> scores in units of 1 / c (c returned): the products, or with a cap (in the form
// CAP) cap_scores, with what `add` adds in these units, less the distance.  Masked keys become -inf; ids: of the keys
// from k0 on, or null.
template <typename T, int NB, Cap CAP, typename F>
__device__ __forceinline__ float score_blocks(const Scoring& a, f16v (&s)[NB], int k0, int pos, bool partial,
                                              const RowMask& m, const int* ids, int lane, F add) {
  const int half = lane >> 5;
  float c = a.scale * kLog2e;
  if (a.cap > 0.f) {
    const float in = a.scale / a.cap;
#pragma unroll
    for (int u = 0; u < NB; ++u) cap_scores<CAP>(s[u], in);
    c = a.cap * (kLog2e * kCapUnits<CAP>);
  }
  add(s);
  if (a.sloped) {
    const float per = -a.slope * kLog2e / c, from = (float)(k0 + 4 * half - pos);
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[u][r] = fmaf(per, fabsf(from + (float)(32 * u + 8 * (r >> 2) + (r & 3))), s[u][r]);
  }
  // Two selects of two instructions each, and only where they decide something: a key past the end has no document.
  if (partial && ids) {
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int4 id = *reinterpret_cast<const int4*>(ids + 32 * u + 8 * g + 4 * half);
        s[u][4 * g] = id.x != m.id ? -INFINITY : s[u][4 * g];
        s[u][4 * g + 1] = id.y != m.id ? -INFINITY : s[u][4 * g + 1];
        s[u][4 * g + 2] = id.z != m.id ? -INFINITY : s[u][4 * g + 2];
        s[u][4 * g + 3] = id.w != m.id ? -INFINITY : s[u][4 * g + 3];
      }
  }
  if (partial && (a.prefixed || !ids)) {
    const int limit = m.limit - k0 - 4 * half;
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 32 * u + 8 * (r >> 2) + (r & 3) >= limit ? -INFINITY : s[u][r];
  }
  return c;
}

// Scores' units, as score_blocks returns them.
template <Cap CAP>
__device__ __forceinline__ float units_of(const Scoring& a) {
  return a.cap > 0.f ? a.cap * (kLog2e * kCapUnits<CAP>) : a.scale * kLog2e;
}

// One step of the running softmax: scores (units log2 / c) -> P as operands; m and l move, returns whether any row's
// outputs must be scaled by alpha first.  l sums P before its rounding: the gradients' P is exact to lse.
template <typename T, int NB>
__device__ __forceinline__ bool softmax_blocks(f16v (&s)[NB], Frag<T> (&p)[NB][2], float c, float& m, float& l,
                                               float& alpha) {
  float top = s[0][0];
#pragma unroll
  for (int u = 0; u < NB; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
  top = half_max(top) * c;
  const bool move = top > m + kLazy;
  const float mn = move ? top : m;
  alpha = move ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
  m = mn;
  const float shift = kLift<T> - mn;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < NB; ++u) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, shift));
      sum[r & 3] += s[u][r];
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) p[u][w] = result_frag<T>(s[u], w);
  }
  l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
  return __any(move);
}

// What rounding 16-bit weights left of them, as operands.  Where a table gets a gradient the weights' products take two or
// three parts: each ds_ij = p_ij (g_i . v_j - delta_i) has an error of p_ij times that of delta_i = g_i . out_i, the same for a
// whole row, which the sums over rows and keys of a bucket do not average out.  With weights rounded once the table's
// gradient is off by 4.6e-4 (2 x 16 heads of 64, 4096 rows on 16x16x16, bf16; fp16 5.8e-5), with two parts by 1.2e-6
// (7e-7), with three, which bf16 has for fp32 tables, by 5e-7; the forward call takes 255, 320 and 384 us.
template <typename T>
__device__ __forceinline__ Frag<T> fine_weights(f16v& s, const Frag<T>& p, int step) {
#pragma unroll
  for (int e = 0; e < 8; ++e) s[8 * step + e] -= (float)p[e];
  return result_frag<T>(s, step);
}

// The values of V that store<true> left out, added to the rows that see their keys.
template <typename T, int ND>
__device__ void add_odd_values(const Args& a, f16v (&o)[ND], const T* v, int k0, unsigned lo, unsigned hi,
                               const RowMask& m, const int* ids, int lane) {
  const int half = fresh<true>(lane) >> 5;  // else the offsets below stay in registers over the caller's loop
  for (int j = 0; j < kTile; ++j) {
    if (((j < 32 ? lo >> j : hi >> (j - 32)) & 1u) == 0u) continue;
    const int key = k0 + j;
    const bool seen = key < m.limit && (!ids || ids[j] == m.id);
    if (!seen) continue;
    const T* row = v + (int64_t)key * a.vl;
#pragma unroll
    for (int b = 0; b < ND; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * b + 8 * g + 4 * half;  // results past the head's values are not stored
        const Vec<float, 4> value = load_as_float<T, 4>(row + min(d, a.d - 4));
#pragma unroll
        for (int r = 0; r < 4; ++r) o[b][4 * g + r] += fabsf(value[r]) < INFINITY ? 0.f : value[r];
      }
  }
}

// Part `split` of [first, last).
__device__ __forceinline__ void split_range(int split, int splits, int& first, int& last) {
  const int per = (last - first + splits - 1) / splits;
  first = min(last, first + split * per);
  last = min(last, first + per);
}

// Four values of an output row, and what their rounding left out.
template <typename T>
__device__ __forceinline__ void store_output(const Args& a, int64_t at, const Vec<float, 4>& v) {
  T* out = static_cast<T*>(a.out) + at;
  store_rounded<T, 4>(out, v);
  if constexpr (sizeof(T) == 2) {
    if (a.rest) {
      const Vec<T, 4> r = __builtin_convertvector(v, Vec<T, 4>);
      const Vec<float, 4> rest = v - __builtin_convertvector(r, Vec<float, 4>);
      if (a.wide_rest) *reinterpret_cast<Vec<float, 4>*>(static_cast<float*>(a.rest) + at) = rest;
      else store_rounded<T, 4>(static_cast<T*>(a.rest) + at, rest);
    }
  }
}

// A lane's O^T results as a row of out, or of the split's sums.
template <typename T, int ND>
__device__ __forceinline__ void write_row(const Args& a, const f16v (&o)[ND], float m, float l, int b, int h, int i,
                                          int split, int lane) {
  const int half = lane >> 5;
  if (a.splits > 1) {
    const int64_t row = (((int64_t)split * a.n + b) * a.hq + h) * a.lq + i;
    const int64_t rows = (int64_t)a.splits * a.n * a.hq * a.lq;
    float* out = a.part + row * (32 * ND);
#pragma unroll
    for (int k = 0; k < ND; ++k)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f4*>(out + 32 * k + 8 * g + 4 * half) =
            f4{o[k][4 * g], o[k][4 * g + 1], o[k][4 * g + 2], o[k][4 * g + 3]};
    if (half == 0) *reinterpret_cast<float2*>(a.part + rows * (32 * ND) + 2 * row) = float2{m, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int64_t out = b * a.ob + h * a.oh + (int64_t)i * a.ol;
#pragma unroll
  for (int k = 0; k < ND; ++k)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * k + 8 * g + 4 * half;
      if (d < a.d) {
        Vec<float, 4> v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = o[k][4 * g + r] * inv;
        store_output<T>(a, out + d, v);
      }
    }
  if (a.lse && half == 0)
    a.lse[((int64_t)b * a.hq + h) * a.lq + i] = l == 0.f ? INFINITY : m + log2f(l) - kLift<T>;
}

extern __shared__ __attribute__((aligned(16))) char bias_values[];  // of a position bias (lay_out_bias)

// The tiled form: a workgroup of four waves takes 128 query rows of a head, 32 a
// wave, and streams K and V through LDS in 64-key tiles: the next tile is loaded
// straight into a second pair of arrays while the current one is multiplied.
// Waves a SIMD that the registers are kept for.  With a bias, 2 x 16 heads of 4096 rows on 16x16x16, bf16: heads of 32 with
// four 187 us (13 registers spill), with three 217; heads of 64 with three 255 (14 spill), with two 264.
template <typename T, int D, int ST>
constexpr int tiled_waves() {
  if (ST == kBias && sizeof(T) == 2 && D < 128) return D == 32 ? 4 : 3;
  return sizeof(T) == 4 && D == 128 ? 1 : 2;
}

template <typename T, int D, Cap CAP, int ST>
__global__ __launch_bounds__(kThreads, (tiled_waves<T, D, ST>())) void attention_kernel(Args a, BiasOf<ST> bias) {
  constexpr int NK = D / 16, ND = D / 32, kMore = ST == 0 ? 0 : ST - kBias;
  typedef Tile<T, D> Lds;
  __shared__ __attribute__((aligned(16))) char kt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char vt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char kt1[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char vt1[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) unsigned words0[kTile];
  __shared__ __attribute__((aligned(16))) unsigned words1[kTile];
  __shared__ unsigned odd[2];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.lq + kRows - 1) / kRows;
  const bool docs = a.qdoc.ids != nullptr;
  int item, block;
  Part part;
  place(blockIdx.x, a.n * a.hq, blocks, docs ? 2 : 1, item, block, part.part);
  if (a.prefixed) block = blocks - 1 - block;  // the longest rows first
  const int b = item / a.hq, h = item % a.hq;
  if (part.part == 1 && !is_mixed(a.qdoc, b, block)) return;
  const int i0 = block * kRows;
  const int i = i0 + 32 * wave + (lane & 31);
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const int* ids = docs ? a.kdoc.ids + (int64_t)b * a.kdoc.stride : nullptr;
  part.first_id = docs ? id_of(a, b, i0) : 0;
  const int own = docs && i < a.lq ? id_of(a, b, i) : 0;
  const bool mine = i < a.lq && (!docs || part.has(own));  // rows of the other part are left to it
  const RowMask mask = {mine ? limit_of(a, i, prefix) : 0, own < 0 || !mine ? -2 : own};
  const int pos = i + a.lk - a.lq;
  const Scoring scoring = scoring_of(a, h);
  const T* q = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + (int64_t)i * a.ql;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + (h / a.group) * a.kh;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + (h / a.group) * a.vh;

  const Meeting meet = meeting<kWaves>(wave, i0, a.lq, [&](int row) { return key_tiles(a, b, row, prefix, &part); });
  int first = meet.all.x, last = meet.all.y;
  split_range(blockIdx.y, a.splits, first, last);

  Frag<T> qf[NK];
#pragma unroll
  for (int s = 0; s < NK; ++s) qf[s] = frag_global(q, s, a.d, lane, mine);
  f16v o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = f16v(0.f);
  float m = kNone, l = 0.f;

  Rows<T, kTile> krows, vrows;
  krows.begin(k, a.kl, first * kTile, a.lk, a.d);
  vrows.begin(v, a.vl, first * kTile, a.lk, a.d);
  unsigned word = 0u;
  if constexpr (ST > 0) {
    word = row_word<kSingle<T, D>>(bias, b, i, a.lq);
    lay_out_bias<kSingle<T, D>, kThreads>(bias, bias_values, h, a.hq, kLog2e / units_of<CAP>(scoring),
                                          t);  // arrive() comes before its use
  }
  typedef Stream<T, D, kTile, kThreads> Load;
  auto fetch = [&](int tile, char* kt, char* vt, unsigned* words) {
    Load::load(kt, krows, t);
    Load::load(vt, vrows, t);
    if constexpr (ST > 0)
      if (wave == 0) load_words(words, (kSingle<T, D> ? bias.key_places : bias.key_codes) + b * bias.key_item, tile * kTile, a.lk, lane);
    krows.next();
    vrows.next();
  };
  // One tile, while the next one is on its way into the other pair of arrays.
  auto step = [&](int tile, char* kt, char* vt, unsigned* words, char* next_kt, char* next_vt, unsigned* next_words) {
    const int k0 = tile * kTile;
    const bool partial = meet.partial(tile);  // some row of the workgroup has a masked key in it
    arrive();
    if (tile + 1 < last) fetch(tile + 1, next_kt, next_vt, next_words);
    if (partial) {
      if (t < 2) odd[t] = 0u;
      __syncthreads();
      Load::clean(vt, odd, t);
      __syncthreads();
    }
    if (meet.skips(tile)) return;
    const int at = fresh<D == 128 && sizeof(T) == 4>(lane);
    f16v s[2] = {f16v(0.f), f16v(0.f)};
    if constexpr (ST > 0)  // without a cap the products are added to the bias
      if (scoring.cap == 0.f) {
#pragma unroll
        for (int u = 0; u < 2; ++u) apply_bias<kSingle<T, D>, true, false, kBiasRows<D>>(s[u], bias_values, word, words + 32 * u, at);
      }
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) s[u] = mma<T>(Lds::along(kt, 32 * u, n, at), qf[n], s[u]);
    // V's first operands are read before the softmax, which covers the latency, as far as registers go.
    constexpr int kEarly = sizeof(T) == 4 ? 0 : D == 128 ? 0 : 2;  // contraction steps
    Frag<T> vf[2][ND];
#pragma unroll
    for (int w = 0; w < kEarly; ++w)
#pragma unroll
      for (int n = 0; n < ND; ++n) vf[w][n] = Lds::down(vt, 16 * w, n, at);
    const int* tile_ids = docs ? ids + k0 : nullptr;
    const float c = score_blocks<T, 2, CAP>(scoring, s, k0, pos, meet.masked(tile), mask, tile_ids, lane, [&](auto& s) {
      if constexpr (ST > 0)
        if (scoring.cap > 0.f) {
#pragma unroll
          for (int u = 0; u < 2; ++u) apply_bias<kSingle<T, D>, true, true, kBiasRows<D>>(s[u], bias_values, word, words + 32 * u, at);
        }
    });
    float alpha;
    Frag<T> p[2][2];
    if (softmax_blocks<T, 2>(s, p, c, m, l, alpha)) {
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        Frag<T> more[kMore > 0 ? kMore : 1];
#pragma unroll
        for (int e = 0; e < kMore; ++e) more[e] = fine_weights<T>(s[u], e == 0 ? p[u][w] : more[e - 1], w);
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          const Frag<T> f = u == 0 && w < kEarly ? vf[w][n] : Lds::down(vt, 32 * u + 16 * w, n, at);
          o[n] = mma<T>(f, p[u][w], o[n]);
#pragma unroll
          for (int e = 0; e < kMore; ++e) o[n] = mma<T>(f, more[e], o[n]);
        }
      }
    if (partial) {
      const unsigned lo = odd[0], hi = odd[1];
      if (lo | hi) add_odd_values<T, ND>(a, o, v, k0, lo, hi, mask, tile_ids, lane);
    }
  };
  if (first < last) fetch(first, kt0, vt0, words0);
  for (int tile = first; tile < last; tile += 2) {
    step(tile, kt0, vt0, words0, kt1, vt1, words1);
    if (tile + 1 < last) step(tile + 1, kt1, vt1, words1, kt0, vt0, words0);
  }
  l = half_sum(l);
  if (mine) write_row<T, ND>(a, o, m, l, b, h, i, blockIdx.y, lane);
}

// The form for few rows: the group * lq <= 32 query rows of a key head are one
// column block, so K and V are read once for all its query heads.  Each wave of a
// workgroup takes every fourth 32-key tile through LDS of its own, without barriers;
// the four results are joined at the end.  Bound by reading K and V: 4 sequences of up
// to 16387 keys, 8 key heads of 128, bf16 (157 MB of visible keys): 39 us, 4 TB/s.
constexpr int kFewTile = 32;

template <typename T, int D>
constexpr int few_lds() {  // bytes; the join takes four 32 x D blocks of fp32 and (m, l) of each
  constexpr int tiles = kWaves * kFewTile * 2 * Tile<T, D>::kRow;
  constexpr int join = kWaves * 32 * (D + 4) * 4;
  return tiles > join ? tiles : join;
}

template <typename T, int D, Cap CAP, int ST>
__global__ __launch_bounds__(kThreads, ST == 0 && sizeof(T) == 4 && D == 64 ? 2 : 1) void attention_few_kernel(
    Args a, BiasOf<ST> bias) {
  constexpr int NK = D / 16, ND = D / 32, kMore = ST == 0 ? 0 : ST - kBias;
  typedef Tile<T, D> Lds;
  __shared__ __attribute__((aligned(16))) unsigned words[kWaves][kFewTile];
  __shared__ __attribute__((aligned(16))) char lds[few_lds<T, D>()];
  __shared__ unsigned odd[kWaves];
  __shared__ float2 state[kWaves][32];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int b = blockIdx.x / a.hk, hk = blockIdx.x % a.hk;
  const int rows = a.group * a.lq, row = min(lane & 31, rows - 1);  // idle columns repeat the last row
  const int h = hk * a.group + row / a.lq, i = row % a.lq;
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const bool docs = a.qdoc.ids != nullptr;
  const int* ids = docs ? a.kdoc.ids + (int64_t)b * a.kdoc.stride : nullptr;
  const int own = docs ? id_of(a, b, i) : 0;
  const RowMask mask = {limit_of(a, i, prefix), own < 0 ? -2 : own};
  const int pos = i + a.lk - a.lq;
  const Scoring scoring = scoring_of(a, h);
  const T* q = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + (int64_t)i * a.ql;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh;
  char* kt = lds + wave * kFewTile * 2 * Lds::kRow;
  char* vt = kt + kFewTile * Lds::kRow;

  const int4 range = key_tiles(a, b, 0, prefix, nullptr);  // lq <= kGrain; tiles of 64 keys
  int first = range.x, last = range.y;
  split_range(blockIdx.y, a.splits, first, last);
  const int end = min(last * kTile, a.lk);

  Frag<T> qf[NK];
#pragma unroll
  for (int s = 0; s < NK; ++s) qf[s] = frag_global(q, s, a.d, lane, true);
  f16v o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = f16v(0.f);
  float m = kNone, l = 0.f;

  // The heads of a group have values of their own, one behind the other.
  unsigned word = 0u, key = 0u;
  const char* values = bias_values;
  if constexpr (ST > 0) {
    word = row_word<kSingle<T, D>>(bias, b, i, a.lq);
    const int bytes = kSingle<T, D> ? 4096 : 4 * bias.values;
    values += (row / a.lq) * bytes;
    for (int g = 0; g < a.group; ++g) {
      lay_out_bias<kSingle<T, D>, kThreads>(bias, bias_values + g * bytes, hk * a.group + g, a.hq,
                                            kLog2e / units_of<CAP>(scoring), t);
      __syncthreads();
    }
  }
  Stream<T, D, kFewTile, 64> ks, vs;
  Rows<T, kFewTile> krows, vrows;
  int k0 = first * kTile + wave * kFewTile;
  auto fetch = [&](int at) {
    krows.begin(k, a.kl, at, a.lk, a.d);
    vrows.begin(v, a.vl, at, a.lk, a.d);
    ks.fetch(krows, lane);
    vs.fetch(vrows, lane);
    if constexpr (ST > 0)
      if (lane < kFewTile) key = key_word<kSingle<T, D>>(bias, b, at + lane, a.lk);
  };
  if (k0 < end) fetch(k0);
  for (; k0 < end; k0 += kWaves * kFewTile) {
    const bool partial = k0 / kTile < range.z || k0 / kTile >= range.w;
    if (lane == 0) odd[wave] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    ks.template store<false>(kt, nullptr, lane);
    if (partial) vs.template store<true>(vt, &odd[wave], lane);
    else vs.template store<false>(vt, nullptr, lane);
    if constexpr (ST > 0)
      if (lane < kFewTile) words[wave][lane] = key;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int next = k0 + kWaves * kFewTile;
    if (next < end) fetch(next);
    f16v s[1] = {f16v(0.f)};
#pragma unroll
    for (int n = 0; n < NK; ++n) s[0] = mma<T>(Lds::along(kt, 0, n, lane), qf[n], s[0]);
    const float c = score_blocks<T, 1, CAP>(scoring, s, k0, pos, partial, mask, docs ? ids + k0 : nullptr, lane,
                                            [&](auto& s) {
                                              if constexpr (ST > 0) apply_bias<kSingle<T, D>, true, true, kBiasRows<D>>(s[0], values, word,
                                                                                             words[wave], lane);
                                            });
    float alpha;
    Frag<T> p[1][2];
    if (softmax_blocks<T, 1>(s, p, c, m, l, alpha)) {
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= alpha;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      Frag<T> more[kMore > 0 ? kMore : 1];
#pragma unroll
      for (int e = 0; e < kMore; ++e) more[e] = fine_weights<T>(s[0], e == 0 ? p[0][w] : more[e - 1], w);
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const Frag<T> f = Lds::down(vt, 16 * w, n, lane);
        o[n] = mma<T>(f, p[0][w], o[n]);
#pragma unroll
        for (int e = 0; e < kMore; ++e) o[n] = mma<T>(f, more[e], o[n]);
      }
    }
    if (partial) {
      const unsigned set = odd[wave];
      if (set) add_odd_values<T, ND>(a, o, v, k0, set, 0u, mask, docs ? ids + k0 : nullptr, lane);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  l = half_sum(l);
  // The join: scaled to the waves' common maximum, summed in the waves' order.
  if (lane < 32) state[wave][lane] = float2{m, l};
  __syncthreads();
  float top = kNone, total = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, state[w][lane & 31].x);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float2 sw = state[w][lane & 31];
    total += sw.y * __builtin_amdgcn_exp2f(sw.x - top);
  }
  const float mine = __builtin_amdgcn_exp2f(m - top);
  float* join = reinterpret_cast<float*>(lds) + wave * 32 * (D + 4);
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f4*>(join + (lane & 31) * (D + 4) + 32 * n + 8 * g + 4 * (lane >> 5)) =
          f4{o[n][4 * g] * mine, o[n][4 * g + 1] * mine, o[n][4 * g + 2] * mine, o[n][4 * g + 3] * mine};
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        sum += *reinterpret_cast<const f4*>(reinterpret_cast<float*>(lds) + (w * 32 + (lane & 31)) * (D + 4) + 32 * n +
                                            8 * g + 4 * (lane >> 5));
#pragma unroll
      for (int r = 0; r < 4; ++r) o[n][4 * g + r] = sum[r];
    }
  if ((lane & 31) < rows) write_row<T, ND>(a, o, top, total, b, h, i, blockIdx.y, lane);
}

// Four joined values of row `at` and, by the thread of its first ones, lse.
template <typename T>
__device__ __forceinline__ void write_joined(const Args& a, int64_t at, int d, const Vec<float, 4>& out, float top,
                                             float total) {
  const int i = (int)(at % a.lq);
  const int64_t bh = at / a.lq;
  const int h = (int)(bh % a.hq);
  const int64_t b = bh / a.hq;
  if (d < a.d) {
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    store_output<T>(a, b * a.ob + h * a.oh + (int64_t)i * a.ol + d, out * inv);
  }
  if (a.lse && d == 0) a.lse[at] = total == 0.f ? INFINITY : top + log2f(total) - kLift<T>;
}

// Joins up to kFewSplits splits: four values of a row a thread, all its loads at once.
constexpr int kFewSplits = 8;

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_join_few_kernel(Args a) {
  const int64_t rows = (int64_t)a.n * a.hq * a.lq;
  const int64_t at = (int64_t)blockIdx.x * (kThreads / (D / 4)) + threadIdx.x / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  if (at >= rows) return;
  const float2* state = reinterpret_cast<const float2*>(a.part + rows * a.splits * D);
  float2 part[kFewSplits];
  f4 value[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    part[s] = float2{kNone, 0.f};
    value[s] = f4{0.f, 0.f, 0.f, 0.f};
    if (s < a.splits) {
      part[s] = state[s * rows + at];
      value[s] = *reinterpret_cast<const f4*>(a.part + (s * rows + at) * D + d);
    }
  }
  float top = kNone, total = 0.f;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) top = fmaxf(top, part[s].x);
  Vec<float, 4> out = Vec<float, 4>(0.f);
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const float w = __builtin_amdgcn_exp2f(part[s].x - top);
    total = fmaf(part[s].y, w, total);
    out += value[s] * w;
  }
  write_joined<T>(a, at, d, out, top, total);
}

// Joins more, one workgroup a row: D / 4 threads hold the values of a split, four each, and the others every
// kThreads / (D / 4)-th split; then in order.  (A thread that walked all splits took 19 us for 128 rows of 32 splits,
// one load after the other; a workgroup a row for 32768 rows of two splits 74 us.)
constexpr int kMostSplits = 64;

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(Args a) {
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ float weight[kMostSplits];
  __shared__ f4 sums[kGroups][kLanes];
  const int64_t rows = (int64_t)a.n * a.hq * a.lq, at = blockIdx.x;
  const int lane = threadIdx.x & 63, d = threadIdx.x % kLanes * 4, group = threadIdx.x / kLanes;
  const float2* state = reinterpret_cast<const float2*>(a.part + rows * a.splits * D);
  const float2 mine = lane < a.splits ? state[lane * rows + at] : float2{kNone, 0.f};
  float top = mine.x;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
  const float w = __builtin_amdgcn_exp2f(mine.x - top);
  float total = mine.y * w;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) total += __shfl_xor(total, m);
  if (threadIdx.x < kMostSplits) weight[threadIdx.x] = w;
  __syncthreads();
  f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = group; s < a.splits; s += kGroups)
    sum += *reinterpret_cast<const f4*>(a.part + (s * rows + at) * D + d) * weight[s];
  sums[group][d / 4] = sum;
  __syncthreads();
  if (group != 0) return;
  Vec<float, 4> out = Vec<float, 4>(0.f);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) out += sums[g][d / 4];
  write_joined<T>(a, at, d, out, top, total);
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
bool few_rows(const ctmr_masked_attention_desc* d) { return (int64_t)(d->q_heads / d->k_heads) * d->lq <= 32; }

// Parts of the keys where the rows alone do not fill the chip: about 512 workgroups, or 256 of the few-row form, of
// at least four 64-key tiles each (two of fp32 heads of 64 and more).  From the shape only, so that a shape's sums have
// one order.  Few rows, bf16, 4 x 8 key heads of 128 values, 16384 keys (268 MB): 49.7 us with 256 workgroups (one a CU
// at a time; 5.4 TB/s), 56 with 384, 51 with 512, 58 with 1024.
int split_count(const ctmr_masked_attention_desc* d) {
  const bool few = few_rows(d);
  const int64_t blocks = (int64_t)d->n * (few ? d->k_heads : d->q_heads * ceil_div(d->lq, kRows));
  const int64_t tiles = ceil_div(d->lk, kTile);
  const int64_t least = d->elem == CTMR_ELEM_F32 && padded(d->head_dim) >= 64 ? 2 : 4;
  const int64_t want = std::max<int64_t>(1, (few ? 256 : 512) / blocks);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, tiles / least, kMostSplits}));
}

template <typename T, int D, Cap CAP, int ST>
void launch_form(const Args& a, const BiasOf<ST>& bias, bool few, hipStream_t st) {
  const unsigned bytes = bias_bytes<T, D>(bias);
  if constexpr (ST > 0) {
    // In the few-row form each head of a group has its values in LDS; where they do not fit the tiled form takes the call.
    constexpr unsigned kRoom = 160 * 1024 - 4096 - few_lds<T, D>();
    few = few && bytes * a.group <= kRoom;
  }
  if (few)
    hipLaunchKernelGGL((attention_few_kernel<T, D, CAP, ST>), dim3(a.n * a.hk, a.splits), dim3(kThreads), bytes * a.group, st,
                       a, bias);
  else
    hipLaunchKernelGGL((attention_kernel<T, D, CAP, ST>),
                       dim3(a.n * a.hq * (unsigned)ceil_div(a.lq, kRows) * (a.qdoc.ids ? 2u : 1u), a.splits), dim3(kThreads),
                       bytes, st, a, bias);
}

template <typename T, int D, int ST>
int launch(const Args& a, const BiasOf<ST>& bias, bool few, hipStream_t st) {
  bool shifted = false;
  if constexpr (sizeof(T) == 2) {  // without a cap too
    shifted = shifted_cap<T>(a.cap);
    if (shifted) launch_form<T, D, kShiftedCap>(a, bias, few, st);
  }
  if (!shifted) launch_form<T, D, kExactCap>(a, bias, few, st);
  const int rc = check_launch("masked_attention");
  if (rc || a.splits == 1) return rc;
  const int64_t rows = (int64_t)a.n * a.hq * a.lq;
  if (a.splits <= kFewSplits)
    hipLaunchKernelGGL((attention_join_few_kernel<T, D>), dim3((unsigned)ceil_div(rows, kThreads / (D / 4))),
                       dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((attention_join_kernel<T, D>), dim3((unsigned)rows), dim3(kThreads), 0, st, a);
  return check_launch("masked_attention_join");
}

}  // namespace
}  // namespace attn
}  // namespace ctmr
