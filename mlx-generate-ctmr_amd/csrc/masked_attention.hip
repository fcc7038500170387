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
#include "masked_attention.hpp"

#include <algorithm>
#include <climits>
#include <cmath>

namespace ctmr {
namespace attn {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRows = 32 * kWaves;  // query rows of a workgroup of the tiled form
constexpr float kLazy = 8.0f;
// fp16 weights are raised by 2^6 (both in O and l): below 2^8 * 2^6 they stay in range, and weights down to
// 2^-20 of the reference keep all their bits.
template <typename T>
constexpr float kLift = std::is_same_v<T, _Float16> ? 6.0f : 0.0f;

// What this lane's row may see: keys below limit whose id is id.
struct RowMask {
  int limit, id;
};

// Raw products of NB 32-key blocks -> scores in units of log2 / c (c returned): with a cap or slopes the scores
// themselves (c = 1), else the products (c = scale log2 e).  Masked keys become -inf; ids: of the keys from k0 on, or
// null.
template <typename T, int NB>
__device__ __forceinline__ float score_blocks(const Args& a, f16v (&s)[NB], int k0, int pos, float slope,
                                              bool partial, const RowMask& m, const int* ids, int lane) {
  const int half = lane >> 5;
  float c = a.scale * kLog2e;
  if (a.cap > 0.f) {
    const float in = a.scale / a.cap, out = a.cap * kLog2e;
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = out * tanh_of<T>(s[u][r] * in);
    c = 1.0f;
  }
  if (a.slopes) {
    const float per = slope * kLog2e;
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = k0 + 32 * u + 8 * (r >> 2) + 4 * half + (r & 3);
        s[u][r] = fmaf(-per, fabsf((float)(pos - j)), s[u][r] * c);
      }
    c = 1.0f;
  }
  if (partial) {
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * u + 8 * g + 4 * half, j = k0 + at;
        int4 id = {m.id, m.id, m.id, m.id};
        if (ids) id = *reinterpret_cast<const int4*>(ids + at);
        if (j >= m.limit || id.x != m.id) s[u][4 * g] = -INFINITY;
        if (j + 1 >= m.limit || id.y != m.id) s[u][4 * g + 1] = -INFINITY;
        if (j + 2 >= m.limit || id.z != m.id) s[u][4 * g + 2] = -INFINITY;
        if (j + 3 >= m.limit || id.w != m.id) s[u][4 * g + 3] = -INFINITY;
      }
  }
  return c;
}

// One step of the running softmax: scores (units log2 / c) -> P; m and l move, returns whether any row's outputs
// must be scaled by alpha first.
template <typename T, int NB>
__device__ __forceinline__ bool softmax_blocks(f16v (&s)[NB], float c, float& m, float& l, float& alpha) {
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
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < NB; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[u][r], c, shift));
      s[u][r] = p;
      sum += p;
    }
  l = l * alpha + sum;
  return __any(move);
}

// The values of V that store<true> left out, added to the rows that see their keys.
template <typename T, int ND>
__device__ void add_odd_values(const Args& a, f16v (&o)[ND], const T* v, int k0, unsigned lo, unsigned hi,
                               const RowMask& m, const int* ids, int lane) {
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
        const int d = 32 * b + 8 * g + 4 * (lane >> 5);  // results past the head's values are not stored
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
// wave, and streams K and V through LDS in 64-key tiles, double-buffered: the loads
// of the next tile are in flight while the current one is multiplied.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void attention_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  constexpr int KS = tile_stride<T, D>(ALONG), VS = tile_stride<T, D>(DOWN);
  __shared__ __attribute__((aligned(16))) T kt[2][kTile * KS];
  __shared__ __attribute__((aligned(16))) T vt[2][kTile * VS];
  __shared__ __attribute__((aligned(16))) int key_ids[2][kTile];
  __shared__ unsigned odd[3][2];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.lq + kRows - 1) / kRows;
  int item, block;
  place(blockIdx.x, a.n * a.hq, blocks, item, block);
  if (a.prefixed) block = blocks - 1 - block;  // the longest rows first
  const int b = item / a.hq, h = item % a.hq;
  const int i0 = block * kRows;
  const int i = i0 + 32 * wave + (lane & 31);
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const bool docs = a.qdoc.ids != nullptr;
  const int* ids = docs ? a.kdoc.ids + (int64_t)b * a.kdoc.stride : nullptr;
  const RowMask mask = {i < a.lq ? limit_of(a, i, prefix) : 0, docs && i < a.lq ? row_id(a, b, i) : -2};
  const int pos = i + a.lk - a.lq;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  const T* q = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + (int64_t)i * a.ql;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + (h / a.group) * a.kh;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + (h / a.group) * a.vh;

  const Meeting meet = meeting<kWaves>(wave, i0, a.lq, [&](int row) { return key_tiles(a, b, row, prefix); });
  int first = meet.all.x, last = meet.all.y;
  split_range(blockIdx.y, a.splits, first, last);

  Frag<T> qf[NK];
#pragma unroll
  for (int s = 0; s < NK; ++s) qf[s] = frag_global(q, s, a.d, lane, i < a.lq);
  f16v o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = f16v(0.f);
  float m = kNone, l = 0.f;

  Stream<T, D, kTile, kThreads> ks, vs;
  bool partial = false;  // of the tile in flight: some row of the workgroup has a masked key in it
  int id = 0;
  auto fetch = [&](int tile) {
    ks.fetch(k, a.kl, tile * kTile, a.lk, a.d, t);
    vs.fetch(v, a.vl, tile * kTile, a.lk, a.d, t);
    partial = meet.partial(tile);
    if (docs && t < kTile) id = ids[tile * kTile + t];
  };
  auto stage = [&](int buf, int slot) {
    ks.template store<false>(kt[buf], KS, nullptr, t);
    if (partial) vs.template store<true>(vt[buf], VS, odd[slot], t);
    else vs.template store<false>(vt[buf], VS, nullptr, t);
    if (docs && t < kTile) key_ids[buf][t] = id;
  };
  if (t < 6) odd[t / 2][t % 2] = 0u;
  if (first < last) {
    fetch(first);
    __syncthreads();
    stage(0, 0);
  }
  int slot = 0;
  for (int tile = first; tile < last; ++tile) {
    const int buf = (tile - first) & 1, k0 = tile * kTile;
    const bool now = partial, more = tile + 1 < last;
    if (more) fetch(tile + 1);
    __syncthreads();
    if (!meet.skips(tile)) {
      f16v s[2] = {f16v(0.f), f16v(0.f)};
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] = mma<T>(frag_along(kt[buf], KS, 32 * u, n, lane), qf[n], s[u]);
      const int* tile_ids = docs ? key_ids[buf] : nullptr;
      const float c = score_blocks<T, 2>(a, s, k0, pos, slope, meet.masked(tile), mask, tile_ids, lane);
      float alpha;
      if (softmax_blocks<T, 2>(s, c, m, l, alpha)) {
#pragma unroll
        for (int n = 0; n < ND; ++n) o[n] *= alpha;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const Frag<T> p = result_frag<T>(s[u], w);
#pragma unroll
          for (int n = 0; n < ND; ++n) o[n] = mma<T>(frag_down(vt[buf], VS, 32 * u + 16 * w, n, lane), p, o[n]);
        }
      if (now) {
        const unsigned lo = odd[slot][0], hi = odd[slot][1];
        if (lo | hi) add_odd_values<T, ND>(a, o, v, k0, lo, hi, mask, tile_ids, lane);
      }
    }
    // Three slots: this tile's is read until the next barrier, the next tile's is set from here on, the one after
    // that was read before this tile's barrier.
    const int next = slot == 2 ? 0 : slot + 1, after = next == 2 ? 0 : next + 1;
    if (t < 2) odd[after][t] = 0u;
    if (more) stage(buf ^ 1, next);
    slot = next;
  }
  l = half_sum(l);
  if (i < a.lq) write_row<T, ND>(a, o, m, l, b, h, i, blockIdx.y, lane);
}

// The form for few rows: the group * lq <= 32 query rows of a key head are one
// column block, so K and V are read once for all its query heads.  Each wave of a
// workgroup takes every fourth 32-key tile through LDS of its own, without barriers;
// the four results are joined at the end.
constexpr int kFewTile = 32;

template <typename T, int D>
constexpr int few_lds() {  // bytes; the join takes four 32 x D blocks of fp32 and (m, l) of each
  constexpr int tiles = kWaves * kFewTile * (tile_stride<T, D>(ALONG) + tile_stride<T, D>(DOWN)) * (int)sizeof(T);
  constexpr int join = kWaves * 32 * (D + 4) * 4;
  return tiles > join ? tiles : join;
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads, 1) void attention_few_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  constexpr int KS = tile_stride<T, D>(ALONG), VS = tile_stride<T, D>(DOWN);
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
  const RowMask mask = {limit_of(a, i, prefix), docs ? row_id(a, b, i) : -2};
  const int pos = i + a.lk - a.lq;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  const T* q = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + (int64_t)i * a.ql;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh;
  T* kt = reinterpret_cast<T*>(lds) + wave * kFewTile * (KS + VS);
  T* vt = kt + kFewTile * KS;

  const int4 range = key_tiles(a, b, 0, prefix);  // lq <= kGrain; tiles of 64 keys
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
  int k0 = first * kTile + wave * kFewTile;
  if (k0 < end) {
    ks.fetch(k, a.kl, k0, a.lk, a.d, lane);
    vs.fetch(v, a.vl, k0, a.lk, a.d, lane);
  }
  for (; k0 < end; k0 += kWaves * kFewTile) {
    const bool partial = k0 / kTile < range.z || k0 / kTile >= range.w;
    if (lane == 0) odd[wave] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    ks.template store<false>(kt, KS, nullptr, lane);
    if (partial) vs.template store<true>(vt, VS, &odd[wave], lane);
    else vs.template store<false>(vt, VS, nullptr, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int next = k0 + kWaves * kFewTile;
    if (next < end) {
      ks.fetch(k, a.kl, next, a.lk, a.d, lane);
      vs.fetch(v, a.vl, next, a.lk, a.d, lane);
    }
    f16v s[1] = {f16v(0.f)};
#pragma unroll
    for (int n = 0; n < NK; ++n) s[0] = mma<T>(frag_along(kt, KS, 0, n, lane), qf[n], s[0]);
    const float c = score_blocks<T, 1>(a, s, k0, pos, slope, partial, mask, docs ? ids + k0 : nullptr, lane);
    float alpha;
    if (softmax_blocks<T, 1>(s, c, m, l, alpha)) {
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= alpha;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Frag<T> p = result_frag<T>(s[0], w);
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] = mma<T>(frag_down(vt, VS, 16 * w, n, lane), p, o[n]);
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

// Joins the splits of a row: 4 values a thread, splits in order.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(Args a) {
  const int64_t rows = (int64_t)a.n * a.hq * a.lq;
  const int64_t at = (int64_t)blockIdx.x * (kThreads * 4 / D) + threadIdx.x / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  if (at >= rows) return;
  const float2* state = reinterpret_cast<const float2*>(a.part + rows * a.splits * D);
  float top = kNone;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, state[s * rows + at].x);
  float total = 0.f;
  Vec<float, 4> sum = Vec<float, 4>(0.f);
  for (int s = 0; s < a.splits; ++s) {
    const float2 sw = state[s * rows + at];
    const float w = __builtin_amdgcn_exp2f(sw.x - top);
    total += sw.y * w;
    sum += *reinterpret_cast<const Vec<float, 4>*>(a.part + (s * rows + at) * D + d) * w;
  }
  const int i = (int)(at % a.lq);
  const int64_t bh = at / a.lq;
  const int h = (int)(bh % a.hq);
  const int64_t b = bh / a.hq;
  if (d < a.d) {
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    store_output<T>(a, b * a.ob + h * a.oh + (int64_t)i * a.ol + d, sum * inv);
  }
  if (a.lse && d == 0) a.lse[at] = total == 0.f ? INFINITY : top + log2f(total) - kLift<T>;
}

// --------------------------------------------------------------------------
// documents: ids of each side, ranges of its tiles and their hulls on the other
// --------------------------------------------------------------------------
struct DocArgs {
  const int* from[2];
  int* ids[2];
  DocTile* tiles[2];
  int4* hull[2];
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

// One wave per kGrain rows: blockIdx = (grain, item, side).
__global__ __launch_bounds__(kTile) void document_hulls_kernel(DocArgs a) {
  const int side = blockIdx.z, b = blockIdx.y, grain = blockIdx.x, lane = threadIdx.x;
  if (grain >= a.grains[side]) return;
  const int i = grain * kGrain + lane % kGrain;
  const int id = i < a.rows[side] ? a.ids[side][(int64_t)b * a.stride[side] + i] : -1;
  DocTile own;
  own.least = i < a.rows[side] ? id : INT_MAX;
  own.most = id;
  own.least_id = id >= 0 ? id : INT_MAX;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    own.least = min(own.least, __shfl_xor(own.least, m));
    own.most = max(own.most, __shfl_xor(own.most, m));
    own.least_id = min(own.least_id, __shfl_xor(own.least_id, m));
  }
  const DocTile* others = a.tiles[1 - side] + (int64_t)b * a.count[1 - side];
  const int count = a.count[1 - side];
  const bool one = own.least == own.most && own.least >= 0;
  int lo = INT_MAX, hi = 0, whole = INT_MAX;
  for (int o = lane; o < count; o += kTile) {
    const DocTile other = others[o];
    if (own.least_id <= other.most && other.least_id <= own.most) {
      lo = min(lo, o);
      hi = max(hi, o + 1);
    }
    if (one && other.least == own.least && other.most == own.least) whole = min(whole, o);
  }
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) {
    lo = min(lo, __shfl_xor(lo, m));
    hi = max(hi, __shfl_xor(hi, m));
    whole = min(whole, __shfl_xor(whole, m));
  }
  // the first run of tiles that hold nothing but this document
  int end = whole == INT_MAX ? 0 : count;
  for (int o = lane; o < end; o += kTile)
    if (o > whole && (others[o].least != own.least || others[o].most != own.least)) end = min(end, o);
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) end = min(end, __shfl_xor(end, m));
  if (lane == 0) a.hull[side][(int64_t)b * a.grains[side] + grain] = int4{lo, hi, whole, end};
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
bool few_rows(const ctmr_masked_attention_desc* d) { return (int64_t)(d->q_heads / d->k_heads) * d->lq <= 32; }

// Parts of the keys where the rows alone do not fill the chip: about 512 workgroups
// (1024 of the few-row form, whose workgroups are bound by the latency of their
// loads), of at least four 64-key tiles each.  From the shape only, so that a shape's
// sums have one order.
int split_count(const ctmr_masked_attention_desc* d) {
  const bool few = few_rows(d);
  const int64_t blocks = (int64_t)d->n * (few ? d->k_heads : d->q_heads * ceil_div(d->lq, kRows));
  const int64_t tiles = ceil_div(d->lk, kTile);
  const int64_t want = std::max<int64_t>(1, (few ? 1024 : 512) / blocks);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, tiles / 4, 64}));
}

template <typename T, int D>
int launch(const Args& a, bool few, hipStream_t st) {
  if (few)
    hipLaunchKernelGGL((attention_few_kernel<T, D>), dim3(a.n * a.hk, a.splits), dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL((attention_kernel<T, D>), dim3(a.n * a.hq * (unsigned)ceil_div(a.lq, kRows), a.splits),
                       dim3(kThreads), 0, st, a);
  const int rc = check_launch("masked_attention");
  if (rc || a.splits == 1) return rc;
  const int64_t rows = (int64_t)a.n * a.hq * a.lq;
  hipLaunchKernelGGL((attention_join_kernel<T, D>), dim3((unsigned)ceil_div(rows, kThreads * 4 / D)), dim3(kThreads), 0,
                     st, a);
  return check_launch("masked_attention_join");
}

}  // namespace

int padded(int head_dim) { return head_dim <= 32 ? 32 : head_dim <= 64 ? 64 : 128; }

static Side side_of(int rows, const int* ids, const void* tiles, const void* hull) {
  Side s = {};
  s.ids = ids;
  s.tiles = static_cast<const DocTile*>(tiles);
  s.hull = static_cast<const int4*>(hull);
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
  const void* qh = take(n * ceil_div(lq, kGrain) * 16);
  const void* kh = take(n * ceil_div(lk, kGrain) * 16);
  q = side_of(lq, qi, qt, qh);
  k = side_of(lk, ki, kt, kh);
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
  if (d->lq > (1 << 28) || d->lk > (1 << 28) ||
      (int64_t)d->n * d->q_heads * ceil_div(std::max(d->lq, d->lk), kTile) > (1ll << 30))
    return fail(CTMR_E_UNSUPPORTED, "too many rows");
  const int bytes = elem_bytes(d->elem);
  for (const int64_t* s : {d->q_strides, d->k_strides, d->v_strides}) {
    if (s[0] < 0 || s[1] < 0 || s[2] < 0 || (s[0] | s[1] | s[2]) * bytes % 16 != 0)
      return fail(CTMR_E_INVALID, "strides must be multiples of 16 bytes and not negative");
    if (s[2] * bytes > (1ll << 31) / kTile - 4096) return fail(CTMR_E_UNSUPPORTED, "row stride too large");
  }
  return CTMR_OK;
}

Args make_args(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const float* slopes,
               const int32_t* prefixes, const void* plan) {
  Args a = {};
  a.q = q, a.k = k, a.v = v, a.slopes = slopes, a.prefixes = prefixes;
  a.n = d->n, a.lq = d->lq, a.lk = d->lk, a.hq = d->q_heads, a.hk = d->k_heads, a.group = d->q_heads / d->k_heads;
  a.d = d->head_dim, a.prefixed = d->prefixed != 0, a.prefix = d->prefix, a.scale = d->scale, a.cap = d->softcap;
  a.qb = d->q_strides[0], a.qh = d->q_strides[1], a.ql = d->q_strides[2];
  a.kb = d->k_strides[0], a.kh = d->k_strides[1], a.kl = d->k_strides[2];
  a.vb = d->v_strides[0], a.vh = d->v_strides[1], a.vl = d->v_strides[2];
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
    a.rows[s] = rows[s], a.stride[s] = sides[s]->stride, a.count[s] = sides[s]->count;
    a.grains[s] = sides[s]->grains;
  }
  const dim3 grid(std::max(a.count[0], a.count[1]), n, 2);
  hipLaunchKernelGGL(document_tiles_kernel, grid, dim3(kTile), 0, (hipStream_t)stream, a);
  const int rc = check_launch("document_tiles");
  if (rc) return rc;
  hipLaunchKernelGGL(document_hulls_kernel, dim3(std::max(a.grains[0], a.grains[1]), n, 2), dim3(kTile), 0, (hipStream_t)stream, a);
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
