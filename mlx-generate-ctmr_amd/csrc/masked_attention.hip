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
// product, half a step of that type on each weight, as the output's own rounding.
//
// Masked places have no effect whatever they hold: masked scores are replaced, and
// in tiles with masked places the values of V that are not finite are zeroed on
// their way into LDS (0 * NaN) and added to the rows that do see them afterwards.
//
// Bound by the softmax's vector operations (five a score: fma, exp, a sum, half a
// maximum, half a conversion) with heads of 32 and 64, by them and the matrix products
// in turn with 128: bf16, 2 x 16 heads of 4096 rows, every key: heads of 32 124 us
// (556 TFLOP/s), of 64 179 (769), of 128 290 (948); fp32, 2 x 8 heads of 2048 rows of
// 32: 84 us, 102 TFLOP/s of the products alone, which run at 153 at best.
#include "masked_attention.hpp"

#include <algorithm>
#include <climits>
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
// CAP) cap_scores, less the distance in these units.  Masked keys become -inf; ids: of the keys from k0 on, or null.
template <typename T, int NB, Cap CAP>
__device__ __forceinline__ float score_blocks(const Scoring& a, f16v (&s)[NB], int k0, int pos, bool partial,
                                              const RowMask& m, const int* ids, int lane) {
  const int half = lane >> 5;
  float c = a.scale * kLog2e;
  if (a.cap > 0.f) {
    const float in = a.scale / a.cap;
#pragma unroll
    for (int u = 0; u < NB; ++u) cap_scores<CAP>(s[u], in);
    c = a.cap * (kLog2e * kCapUnits<CAP>);
  }
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
      store_rounded<T, 4>(static_cast<T*>(a.rest) + at, v - __builtin_convertvector(r, Vec<float, 4>));
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

// The tiled form: a workgroup of four waves takes 128 query rows of a head, 32 a
// wave, and streams K and V through LDS in 64-key tiles: the next tile is loaded
// straight into a second pair of arrays while the current one is multiplied.
template <typename T, int D, Cap CAP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && D == 128 ? 1 : 2) void attention_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  typedef Tile<T, D> Lds;
  __shared__ __attribute__((aligned(16))) char kt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char vt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char kt1[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char vt1[kTile * Lds::kRow];
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
  typedef Stream<T, D, kTile, kThreads> Load;
  auto fetch = [&](char* kt, char* vt) {
    Load::load(kt, krows, t);
    Load::load(vt, vrows, t);
    krows.next();
    vrows.next();
  };
  // One tile, while the next one is on its way into the other pair of arrays.
  auto step = [&](int tile, char* kt, char* vt, char* next_kt, char* next_vt) {
    const int k0 = tile * kTile;
    const bool partial = meet.partial(tile);  // some row of the workgroup has a masked key in it
    arrive();
    if (tile + 1 < last) fetch(next_kt, next_vt);
    if (partial) {
      if (t < 2) odd[t] = 0u;
      __syncthreads();
      Load::clean(vt, odd, t);
      __syncthreads();
    }
    if (meet.skips(tile)) return;
    const int at = fresh<D == 128 && sizeof(T) == 4>(lane);
    f16v s[2] = {f16v(0.f), f16v(0.f)};
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
    const float c = score_blocks<T, 2, CAP>(scoring, s, k0, pos, meet.masked(tile), mask, tile_ids, lane);
    float alpha;
    Frag<T> p[2][2];
    if (softmax_blocks<T, 2>(s, p, c, m, l, alpha)) {
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int n = 0; n < ND; ++n)
          o[n] = mma<T>(u == 0 && w < kEarly ? vf[w][n] : Lds::down(vt, 32 * u + 16 * w, n, at), p[u][w], o[n]);
    if (partial) {
      const unsigned lo = odd[0], hi = odd[1];
      if (lo | hi) add_odd_values<T, ND>(a, o, v, k0, lo, hi, mask, tile_ids, lane);
    }
  };
  if (first < last) fetch(kt0, vt0);
  for (int tile = first; tile < last; tile += 2) {
    step(tile, kt0, vt0, kt1, vt1);
    if (tile + 1 < last) step(tile + 1, kt1, vt1, kt0, vt0);
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

template <typename T, int D, Cap CAP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && D == 64 ? 2 : 1) void attention_few_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  typedef Tile<T, D> Lds;
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

  Stream<T, D, kFewTile, 64> ks, vs;
  Rows<T, kFewTile> krows, vrows;
  int k0 = first * kTile + wave * kFewTile;
  auto fetch = [&](int at) {
    krows.begin(k, a.kl, at, a.lk, a.d);
    vrows.begin(v, a.vl, at, a.lk, a.d);
    ks.fetch(krows, lane);
    vs.fetch(vrows, lane);
  };
  if (k0 < end) fetch(k0);
  for (; k0 < end; k0 += kWaves * kFewTile) {
    const bool partial = k0 / kTile < range.z || k0 / kTile >= range.w;
    if (lane == 0) odd[wave] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    ks.template store<false>(kt, nullptr, lane);
    if (partial) vs.template store<true>(vt, &odd[wave], lane);
    else vs.template store<false>(vt, nullptr, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int next = k0 + kWaves * kFewTile;
    if (next < end) fetch(next);
    f16v s[1] = {f16v(0.f)};
#pragma unroll
    for (int n = 0; n < NK; ++n) s[0] = mma<T>(Lds::along(kt, 0, n, lane), qf[n], s[0]);
    const float c = score_blocks<T, 1, CAP>(scoring, s, k0, pos, partial, mask, docs ? ids + k0 : nullptr, lane);
    float alpha;
    Frag<T> p[1][2];
    if (softmax_blocks<T, 1>(s, p, c, m, l, alpha)) {
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= alpha;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] = mma<T>(Lds::down(vt, 16 * w, n, lane), p[0][w], o[n]);
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
// documents: ids of each side, ranges of its tiles and their hulls on the other
// --------------------------------------------------------------------------
struct DocArgs {
  const int* from[2];
  int* ids[2];
  DocTile* tiles[2];
  int4* hull[2];
  int* mixed[2];
  int rows[2], stride[2], count[2], grains[2];
};

// One wave per tile: blockIdx = (tile, item, side).
__global__ __launch_bounds__(kTile) void document_tiles_kernel(DocArgs a) {
  const int side = blockIdx.z, b = blockIdx.y, tile = blockIdx.x, lane = threadIdx.x;
  if (tile >= a.count[side]) return;
  const int i = tile * kTile + lane;
  const bool real = i < a.rows[side];
  const int id = real ? max(a.from[side][(int64_t)b * a.rows[side] + i], -1) : -1;
  a.ids[side][(int64_t)b * a.stride[side] + i] = id;
  int least = real ? id : INT_MAX, most = id, least_id = id >= 0 ? id : INT_MAX;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    least = min(least, __shfl_xor(least, m));
    most = max(most, __shfl_xor(most, m));
    least_id = min(least_id, __shfl_xor(least_id, m));
  }
  if (lane == 0) a.tiles[side][(int64_t)b * a.count[side] + tile] = DocTile{least, most, least_id, 0};
}

// Tiles of a side [x, y) that may hold ids least .. most, and the first run [z, w) of tiles that hold only the one
// id, for least = most >= 0.
__device__ __forceinline__ int4 document_run(const DocArgs& a, int side, int b, int lane, int least, int most) {
  const DocTile* tiles = a.tiles[side] + (int64_t)b * a.count[side];
  const int count = a.count[side];
  const bool one = least == most;
  int4 run = {INT_MAX, 0, INT_MAX, 0};
  if (most < 0 || least > most) return run;
  for (int o = lane; o < count; o += kTile) {
    const DocTile tile = tiles[o];
    if (least <= tile.most && tile.least_id <= most) {
      run.x = min(run.x, o);
      run.y = max(run.y, o + 1);
    }
    if (one && tile.least == least && tile.most == least) run.z = min(run.z, o);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    run.x = min(run.x, __shfl_xor(run.x, m));
    run.y = max(run.y, __shfl_xor(run.y, m));
    run.z = min(run.z, __shfl_xor(run.z, m));
  }
  int end = run.z == INT_MAX ? 0 : count;
  for (int o = lane; o < end; o += kTile)
    if (o > run.z && (tiles[o].least != least || tiles[o].most != least)) end = min(end, o);
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) end = min(end, __shfl_xor(end, m));
  run.w = end;
  return run;
}

// One wave per kGrain rows: blockIdx = (grain, item, side).
__global__ __launch_bounds__(kTile) void document_hulls_kernel(DocArgs a) {
  const int side = blockIdx.z, b = blockIdx.y, grain = blockIdx.x, lane = threadIdx.x;
  if (grain >= a.grains[side]) return;
  if (grain % 4 == 0) {
    const int* ids = a.ids[side] + (int64_t)b * a.stride[side];
    bool other = false;
#pragma unroll
    for (int r = lane; r < kBlockRows; r += kTile) {
      const int row = grain * kGrain + r;
      other |= row < a.rows[side] && ids[row] != ids[grain * kGrain];
    }
    other = __any(other);
    if (lane == 0) a.mixed[side][(int64_t)b * ((a.grains[side] + 3) / 4) + grain / 4] = other;
  }
  const int i = grain * kGrain + lane % kGrain;
  const int id = i < a.rows[side] ? a.ids[side][(int64_t)b * a.stride[side] + i] : -1;
  // The first row's document, and the range of the other rows' ids, padding aside: which tiles may hold them, and
  // the first run of tiles that hold nothing else.
  const int first = __shfl(id, 0);
  int least = id >= 0 && id != first ? id : INT_MAX, most = id != first ? id : -1;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    least = min(least, __shfl_xor(least, m));
    most = max(most, __shfl_xor(most, m));
  }
  const bool padded = __any(i < a.rows[side] && id < 0 && first >= 0);
  const int4 own = document_run(a, 1 - side, b, lane, first, first);
  int4 rest = document_run(a, 1 - side, b, lane, least, most);
  if (padded) rest.z = INT_MAX, rest.w = 0;  // the padding goes with the other documents and sees none of their tiles
  if (lane == 0) {
    int4* hull = a.hull[side] + 3 * ((int64_t)b * a.grains[side] + grain);
    hull[0] = own;
    hull[1] = rest;
    // padding among the rows is as good as another document that no tile holds, so no tile is whole for the rest
    hull[2] = least <= most ? int4{padded ? -1 : least, most, 0, 0} : padded ? int4{-1, -1, 0, 0} : int4{1, 0, 0, 0};
  }
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

template <typename T, int D, Cap CAP>
void launch_form(const Args& a, bool few, hipStream_t st) {
  if (few)
    hipLaunchKernelGGL((attention_few_kernel<T, D, CAP>), dim3(a.n * a.hk, a.splits), dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((attention_kernel<T, D, CAP>),
                       dim3(a.n * a.hq * (unsigned)ceil_div(a.lq, kRows) * (a.qdoc.ids ? 2u : 1u), a.splits), dim3(kThreads),
                       0, st, a);
}

template <typename T, int D>
int launch(const Args& a, bool few, hipStream_t st) {
  bool shifted = false;
  if constexpr (sizeof(T) == 2) {  // without a cap too
    shifted = shifted_cap<T>(a.cap);
    if (shifted) launch_form<T, D, kShiftedCap>(a, few, st);
  }
  if (!shifted) launch_form<T, D, kExactCap>(a, few, st);
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

int padded(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }

static Side side_of(int rows, const int* ids, const void* tiles, const void* hull, const int* mixed) {
  Side s = {};
  s.ids = ids;
  s.tiles = static_cast<const DocTile*>(tiles);
  s.hull = static_cast<const int4*>(hull);
  s.mixed = mixed;
  s.count = (int)ceil_div(rows, kTile);
  s.stride = s.count * kTile;
  s.grains = (int)ceil_div(rows, kGrain);
  return s;
}

// A plan's parts: ids of both sides, tiles of both, hulls of both.
static void plan_parts(int32_t n, int32_t lq, int32_t lk, char* base, Side& q, Side& k, int64_t* bytes) {
  const int64_t nq = ceil_div(lq, kTile), nk = ceil_div(lk, kTile);
  int64_t at = 0;
  auto take = [&](int64_t size) {
    const int64_t here = at;
    at += size;
    return base ? base + here : nullptr;
  };
  const int* qi = (const int*)take(n * nq * kTile * 4);
  const int* ki = (const int*)take(n * nk * kTile * 4);
  const void* qt = take(n * nq * (int64_t)sizeof(DocTile));
  const void* kt = take(n * nk * (int64_t)sizeof(DocTile));
  const void* qh = take(n * ceil_div(lq, kGrain) * 48);
  const void* kh = take(n * ceil_div(lk, kGrain) * 48);
  const int* qm = (const int*)take(n * ceil_div(lq, kBlockRows) * 4);
  const int* km = (const int*)take(n * ceil_div(lk, kBlockRows) * 4);
  q = side_of(lq, qi, qt, qh, qm);
  k = side_of(lk, ki, kt, kh, km);
  if (bytes) *bytes = at;
}

int check_desc(const ctmr_masked_attention_desc* d) {
  if (!d) return fail(CTMR_E_INVALID, "null descriptor");
  if (d->n <= 0 || d->lq <= 0 || d->lk <= 0 || d->q_heads <= 0 || d->k_heads <= 0)
    return fail(CTMR_E_INVALID, "non-positive dimension");
  if (d->q_heads % d->k_heads != 0) return fail(CTMR_E_INVALID, "query heads must be a multiple of key heads");
  if (!valid_elem(d->elem)) return fail(CTMR_E_INVALID, "bad element type");
  if (d->head_dim <= 0 || d->head_dim % 8 != 0 || d->head_dim > 128)
    return fail(CTMR_E_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128");
  if (!(d->scale > 0.f) || !(d->scale < INFINITY) || !(d->softcap >= 0.f) || !(d->softcap < INFINITY))
    return fail(CTMR_E_INVALID, "scale must be positive, softcap not negative, both finite");
  if (d->softcap > 0.f && !(d->scale / d->softcap < 1e30f))
    return fail(CTMR_E_INVALID, "softcap too small for the scale");
  if (d->softcap > 1e30f || (d->softcap > 0.f && d->scale / d->softcap < 1e-30f))  // fp32 ends not far above
    return fail(CTMR_E_INVALID, "softcap too large for the scale");
  if (d->lq > (1 << 28) || d->lk > (1 << 28) ||
      (int64_t)d->n * d->q_heads * ceil_div(std::max(d->lq, d->lk), kTile) > (1ll << 23))  // 2^32 threads
    return fail(CTMR_E_UNSUPPORTED, "too many rows");
  int rc = check_strides(d, d->q_strides, d->lq);
  if (!rc) rc = check_strides(d, d->k_strides, d->lk);
  return rc ? rc : check_strides(d, d->v_strides, d->lk);
}

// Rows may not overlap: the kernels take what lies past the last one as out of range.
int check_strides(const ctmr_masked_attention_desc* d, const int64_t* s, int rows) {
  const int bytes = elem_bytes(d->elem);
  if (s[0] < 0 || s[1] < 0 || s[2] < 0 || (s[0] | s[1] | s[2]) * bytes % 16 != 0)
    return fail(CTMR_E_INVALID, "strides must be multiples of 16 bytes and not negative");
  if (rows > 1 && s[2] < d->head_dim) return fail(CTMR_E_INVALID, "rows overlap");
  if (s[2] * bytes > (1ll << 30) / kTile - 4096) return fail(CTMR_E_UNSUPPORTED, "row stride too large");
  return CTMR_OK;
}

int64_t row_stride(const int64_t* s, int rows, int head_dim) { return rows > 1 ? s[2] : head_dim; }

Args make_args(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const float* slopes,
               const int32_t* prefixes, const void* plan) {
  Args a = {};
  a.q = q, a.k = k, a.v = v, a.slopes = slopes, a.prefixes = prefixes;
  a.n = d->n, a.lq = d->lq, a.lk = d->lk, a.hq = d->q_heads, a.hk = d->k_heads, a.group = d->q_heads / d->k_heads;
  a.d = d->head_dim, a.prefixed = d->prefixed != 0, a.prefix = d->prefix, a.scale = d->scale, a.cap = d->softcap;
  a.qb = d->q_strides[0], a.qh = d->q_strides[1], a.ql = row_stride(d->q_strides, d->lq, d->head_dim);
  a.kb = d->k_strides[0], a.kh = d->k_strides[1], a.kl = row_stride(d->k_strides, d->lk, d->head_dim);
  a.vb = d->v_strides[0], a.vh = d->v_strides[1], a.vl = row_stride(d->v_strides, d->lk, d->head_dim);
  a.splits = 1;
  if (plan) plan_parts(d->n, d->lq, d->lk, (char*)plan, a.qdoc, a.kdoc, nullptr);
  return a;
}

}  // namespace attn
}  // namespace ctmr

using namespace ctmr;
using namespace ctmr::attn;

extern "C" {

int64_t ctmr_documents_bytes(int32_t n, int32_t lq, int32_t lk) {
  if (n <= 0 || lq <= 0 || lk <= 0) return fail(CTMR_E_INVALID, "non-positive dimension");
  if (n > 65535 || lq > (1 << 28) || lk > (1 << 28)) return fail(CTMR_E_UNSUPPORTED, "too many rows");
  Side q, k;
  int64_t bytes = 0;
  plan_parts(n, lq, lk, nullptr, q, k, &bytes);
  return bytes;
}

int ctmr_documents(int32_t n, int32_t lq, int32_t lk, const int32_t* query_ids, const int32_t* key_ids, void* plan,
                   size_t plan_bytes, void* stream) {
  const int64_t need = ctmr_documents_bytes(n, lq, lk);
  if (need < 0) return (int)need;
  if (!query_ids || !key_ids || !plan) return fail(CTMR_E_INVALID, "null pointer");
  if ((int64_t)plan_bytes < need || ((uintptr_t)plan & 15) != 0)
    return fail(CTMR_E_WORKSPACE, "document plan too small or not on a 16-byte boundary");
  Side q, k;
  plan_parts(n, lq, lk, (char*)plan, q, k, nullptr);
  DocArgs a = {};
  a.from[0] = query_ids, a.from[1] = key_ids;
  const Side* sides[2] = {&q, &k};
  const int rows[2] = {lq, lk};
  for (int s = 0; s < 2; ++s) {
    a.ids[s] = const_cast<int*>(sides[s]->ids);
    a.tiles[s] = const_cast<DocTile*>(sides[s]->tiles);
    a.hull[s] = const_cast<int4*>(sides[s]->hull);
    a.mixed[s] = const_cast<int*>(sides[s]->mixed);
    a.rows[s] = rows[s], a.stride[s] = sides[s]->stride, a.count[s] = sides[s]->count;
    a.grains[s] = sides[s]->grains;
  }
  const dim3 grid(std::max(a.count[0], a.count[1]), n, 2);
  hipLaunchKernelGGL(document_tiles_kernel, grid, dim3(kTile), 0, (hipStream_t)stream, a);
  const int rc = check_launch("document_tiles");
  if (rc) return rc;
  hipLaunchKernelGGL(document_hulls_kernel, dim3(std::max(a.grains[0], a.grains[1]), n, 2), dim3(kTile), 0,
                     (hipStream_t)stream, a);
  return check_launch("document_hulls");
}

int64_t ctmr_masked_attention_workspace_bytes(const ctmr_masked_attention_desc* d) {
  const int rc = check_desc(d);
  if (rc) return rc;
  const int64_t splits = split_count(d);
  return splits == 1 ? 0 : splits * d->n * d->q_heads * d->lq * (padded(d->head_dim) + 2) * 4;
}

int ctmr_masked_attention(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v,
                          const float* slopes, const int32_t* prefixes, const void* plan, void* out, void* rest,
                          float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t need = ctmr_masked_attention_workspace_bytes(d);
  if (need < 0) return (int)need;
  if (!q || !k || !v || !out) return fail(CTMR_E_INVALID, "null pointer");
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest | (uintptr_t)plan) & 15) !=
      0)
    return fail(CTMR_E_INVALID, "q, k, v, out, rest and the document plan must start on 16-byte boundaries");
  if ((d->out_strides[0] | d->out_strides[1] | d->out_strides[2]) % 4 != 0)
    return fail(CTMR_E_INVALID, "strides of out must be multiples of 4 values");
  if (need > 0 && ((int64_t)workspace_bytes < need || !workspace || ((uintptr_t)workspace & 15) != 0)) {
    set_error("attention workspace: %zu bytes given, %lld needed on a 16-byte boundary", workspace_bytes,
              (long long)need);
    return CTMR_E_WORKSPACE;
  }
  Args a = make_args(d, q, k, v, slopes, prefixes, plan);
  a.out = out, a.rest = rest, a.lse = lse, a.part = (float*)workspace, a.splits = split_count(d);
  a.ob = d->out_strides[0], a.oh = d->out_strides[1], a.ol = d->out_strides[2];
  const bool few = few_rows(d);
  hipStream_t st = (hipStream_t)stream;
#define CTMR_ATTENTION_CASE(T)                          \
  switch (padded(d->head_dim)) {                        \
    case 32: return launch<T, 32>(a, few, st);          \
    case 64: return launch<T, 64>(a, few, st);          \
    default: return launch<T, 128>(a, few, st);         \
  }
  if (d->elem == CTMR_ELEM_F32) CTMR_ATTENTION_CASE(float)
  if (d->elem == CTMR_ELEM_BF16) CTMR_ATTENTION_CASE(__bf16)
  CTMR_ATTENTION_CASE(_Float16)
#undef CTMR_ATTENTION_CASE
}

}  // extern "C"
