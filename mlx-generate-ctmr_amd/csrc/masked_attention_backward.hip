// Gradients of the masked attention (masked_attention.hip), for fp32, bf16 and fp16.
//
// With p_ij = 2^(s2_ij - lse_i) recomputed from q, k and lse, g = dout:
//   dv_j = sum_i p_ij g_i
//   ds_ij = p_ij (g_i . v_j - delta_i) (1 - t_ij^2),  delta_i = g_i . out_i,
//           t = tanh(scale q_i . k_j / cap), 0 without a cap
// delta takes out before its rounding (out + rest, as the forward call left it): with
// few visible keys g . v_j - delta_i is small beside both, and out's half steps would
// be the largest error of dq and dk.
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i
// sums over i running over all query heads that share the key head.
//
// Two kernels, each a stream of one side's tiles through LDS against 128 rows of
// the other in registers: queries stay and keys stream for dq (and delta, which it
// leaves for the other), keys stay and queries stream for dk and dv.  That is seven
// products for the five of the formulas (scores and g . v twice), but no additions in
// memory: each sum has one order, and the gradients are bit-identical run to run.  Where
// the blocks of 128 rows do not fill the chip, each block's stream is cut into parts
// whose fp32 sums a third kernel adds in order.  p and ds are rounded to the operands'
// type for their products, half a step of it on each term of an fp32 sum.
//
// Bound by the matrix products and, at their side, the exponentials: 2 x 16 heads of
// 4096 rows, every key, bf16, both kernels: heads of 32 327 us, of 64 505 (680 TFLOP/s
// of the five products, 950 of the seven), of 128 990; fp16 378, 568, 1147 (the powers of
// two below: two operations a score in dk and dv, half a one in dq); fp32, 2 x 8 heads of
// 2048 rows of 32: 252 (119 of the seven, where a library product of 8192^3 reaches 153).
//
// fp16's range is far smaller than what ds spans, so every row of dq and every key of
// dk (a lane's column) has a power of two of its own that ds is multiplied by: the sums
// start with 2^40 and move down, like a running maximum, when a ds passes 2^15.  Values
// of ds down to 2^-38 of the largest that the row or key has met count, whatever other
// rows, heads and documents hold.  p is raised by 2^15.  All comes out of the sums again
// at the end, exactly.
#include "masked_attention.hpp"

#include <algorithm>
#include <cmath>

namespace ctmr {
namespace attn {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kOwn = kBlockRows;  // rows that a workgroup keeps in registers
static_assert(kOwn == 32 * kWaves && kOwn == 4 * kGrain, "32 rows a wave");

// What dq and dk are multiplied by at the end.
template <Cap CAP>
__host__ __device__ __forceinline__ float ds_scale(const Args& a) {
  return a.scale * (CAP == kNoCap ? 1.0f : kCapSlope<CAP>);
}

template <typename T>
constexpr bool kHalf = std::is_same_v<T, _Float16>;
constexpr float kRaise = 15.0f;  // of p, in log2
// log2 of what fp16's ds are multiplied by at first: those that need more (below 2^-54, where they lose bits) are nothing
// in a gradient, |ds k| < 2^-38, and the largest, below 2^40, stay far from fp32's end.
template <typename T>
constexpr float kDsRaise = kHalf<T> ? 40.0f : 0.0f;

// Keeps a lane's ds, multiplied by 2^raise, in fp16's range, its sums with them: a ds past 2^15 takes the largest to
// [2^13, 2^14).  What is not finite moves nothing.  The lanes of a column, l and l + 32, move together.
// ACC: the sums live in accumulation registers, and are taken out of them nowhere but here (left to itself the compiler
// moves dk's 64 to and fro in each block: 2 x 16 heads of 4096 rows of 128, dk and dv 787 us for 740).
template <bool ACC, int ND>
__device__ __forceinline__ void keep_in_range(f16v& ds, f16v (&sums)[ND], float& raise) {
  float top = fabsf(ds[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
  top = half_max(top);
  const bool over = top > 32768.0f && top < INFINITY;
  if (__any(over)) {
    const int down = over ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
    const float factor = __builtin_ldexpf(1.0f, -down);
    ds *= factor;
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      if constexpr (ACC) asm("" : "+a"(sums[n]));
      sums[n] *= factor;
      if constexpr (ACC) asm("" : "+a"(sums[n]));
    }
    raise -= (float)down;
  }
}

// Products of a 32 x 32 block -> log2 scores in units of 1 / c (c returned).  Row r of a lane is `at` + 8 (r / 4) + r
// % 4; `x` is where the distance to it is zero.  With CAP g . v - delta, in `ds`, is multiplied by 1 - t^2
// (in units of kCapSlope).  (As a branch on the cap the factor was 48 instructions of 145 a block for every call: the
// compiler computes and selects.)
template <typename T, Cap CAP>
__device__ __forceinline__ float scores(const Scoring& a, f16v& s, f16v& ds, int at, int x) {
  float c = a.scale * kLog2e;
  if constexpr (CAP != kNoCap) {
    cap_scores<CAP>(s, a.scale / a.cap);
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= cap_slope<CAP>(s[r]);
    c = a.cap * (kLog2e * kCapUnits<CAP>);
  }
  if (a.sloped) {
    const float per = -a.slope * kLog2e / c, from = (float)(at - x);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(per, fabsf(from + (float)(8 * (r >> 2) + (r & 3))), s[r]);
  }
  return c;
}

// Takes fp16's 2^raise out of the sums.
template <typename T, int ND>
__device__ __forceinline__ void lower(f16v (&sums)[ND], float raise) {
  if constexpr (kHalf<T>) {
    const float factor = __builtin_ldexpf(1.0f, -(int)raise);
#pragma unroll
    for (int n = 0; n < ND; ++n) sums[n] *= factor;
  }
}

template <typename T, int ND>
__device__ __forceinline__ void write_gradient(T* out, const f16v (&g)[ND], float scale, int d, int lane) {
#pragma unroll
  for (int k = 0; k < ND; ++k)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 32 * k + 8 * q + 4 * (lane >> 5);
      if (at < d) {
        Vec<float, 4> v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = g[k][4 * q + r] * scale;
        store_rounded<T, 4>(out + at, v);
      }
    }
}

// The first of `count` steps of part `split` of `splits`, and the one past its last.
__device__ __forceinline__ int2 split_steps(int count, int split, int splits) {
  const int per = (count + splits - 1) / splits, first = min(count, split * per);
  return {first, min(count, first + per)};
}

// Waves a SIMD that the registers are kept for.  16-bit, 2 x 16 heads of 4096 rows, both kernels: heads of 32 with four
// 327 us (a few registers spill), with three 351; heads of 64 with three for dk and dv too (20 spill) 577 us, with two
// there 505.
template <typename T, int D>
constexpr int dq_waves() {
  return D * sizeof(T) >= 512 ? 1 : D * sizeof(T) == 64 ? 4 : D * sizeof(T) == 128 ? 3 : 2;
}

// dq and delta: 128 query rows of a head, key tiles streaming.
template <typename T, int D, Cap CAP>
__global__ __launch_bounds__(kThreads, (dq_waves<T, D>())) void attention_dq_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  typedef Tile<T, D> Lds;
  __shared__ __attribute__((aligned(16))) char kt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char vt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char kt1[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char vt1[kTile * Lds::kRow];
  __shared__ unsigned odd[2];
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.lq + kOwn - 1) / kOwn;
  const bool docs = a.qdoc.ids != nullptr;
  int item, block;
  Part part;
  place(blockIdx.x, a.n * a.hq, blocks, docs ? 2 : 1, item, block, part.part);
  if (a.prefixed) block = blocks - 1 - block;
  const int b = item / a.hq, h = item % a.hq;
  if (part.part == 1 && !is_mixed(a.qdoc, b, block)) return;
  const int i0 = block * kOwn;
  const int i = i0 + 32 * wave + (lane & 31);
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const int* ids = docs ? a.kdoc.ids + (int64_t)b * a.kdoc.stride : nullptr;
  part.first_id = docs ? id_of(a, b, i0) : 0;
  const int own = docs && i < a.lq ? id_of(a, b, i) : 0;
  const bool real = i < a.lq && (!docs || part.has(own));  // rows of the other part are left to it
  const int limit = real ? limit_of(a, i, prefix) : 0, id = own < 0 || !real ? -2 : own;
  const int pos = i + a.lk - a.lq;
  const Scoring scoring = scoring_of(a, h);
  const int64_t stat = ((int64_t)b * a.hq + h) * a.lq + i;
  const T* q = static_cast<const T*>(a.q) + b * a.qb + h * a.qh + (int64_t)i * a.ql;
  const T* g = static_cast<const T*>(a.dout) + b * a.gb + h * a.gh + (int64_t)i * a.gl;
  const T* out = static_cast<const T*>(a.out) + b * a.ob + h * a.oh + (int64_t)i * a.ol;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + (h / a.group) * a.kh;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + (h / a.group) * a.vh;

  Frag<T> qf[NK], gf[NK];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < NK; ++s) {
    qf[s] = frag_global(q, s, a.d, lane, real);
    gf[s] = frag_global(g, s, a.d, lane, real);
    const Frag<T> of = frag_global(out, s, a.d, lane, real);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[s][e], (float)of[e], delta);
    if constexpr (sizeof(T) == 2) {
      if (a.rest) {
        const T* rest = static_cast<const T*>(a.rest) + b * a.ob + h * a.oh + (int64_t)i * a.ol;
        const Frag<T> rf = frag_global(rest, s, a.d, lane, real);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[s][e], (float)rf[e], delta);
      }
    }
  }
  delta = half_sum(delta);
  if (real && half == 0 && blockIdx.y == 0) a.delta[stat] = -delta;
  if (!a.dq) return;
  const float lse = real ? a.lse[stat] : INFINITY;
  float raise = kDsRaise<T>;
  f16v dq[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) dq[n] = f16v(0.f);

  const Meeting meet = meeting<kWaves>(wave, i0, a.lq, [&](int row) { return key_tiles(a, b, row, prefix, &part); });
  const int2 mine = split_steps(meet.all.y - meet.all.x, blockIdx.y, a.splits);
  const int first = meet.all.x + mine.x, last = meet.all.x + mine.y;
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
    const bool partial = meet.partial(tile);
    arrive();
    if (tile + 1 < last) fetch(next_kt, next_vt);
    if (partial) {
      if (t < 2) odd[t] = 0u;
      __syncthreads();
      Load::clean(kt, odd, t);
      __syncthreads();
    }
    if (meet.skips(tile)) return;
    const int la = fresh<D == 128 && sizeof(T) == 2 && CAP != kNoCap>(lane);
    const bool masked = meet.masked(tile) || (partial && (odd[0] | odd[1]) != 0u);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f16v s = f16v(0.f), ds = f16v(-delta);
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        s = mma<T>(Lds::along(kt, 32 * u, n, la), qf[n], s);
        ds = mma<T>(Lds::along(vt, 32 * u, n, la), gf[n], ds);
      }
      const int at = k0 + 32 * u + 4 * half;
      const float c = scores<T, CAP>(scoring, s, ds, at, pos);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= __builtin_amdgcn_exp2f(fmaf(s[r], c, kHalf<T> ? raise - lse : -lse));
      if (masked) {
        // a visible key whose values were zeroed in LDS because they are not finite: no gradient is
        const unsigned set = partial ? odd[u] >> (4 * half) : 0u;
        if (set)
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = (set >> (8 * (r >> 2) + (r & 3))) & 1u ? NAN : ds[r];
        if (docs)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int4 other = *reinterpret_cast<const int4*>(ids + k0 + 32 * u + 4 * half + 8 * w);
            ds[4 * w] = other.x != id ? 0.f : ds[4 * w];
            ds[4 * w + 1] = other.y != id ? 0.f : ds[4 * w + 1];
            ds[4 * w + 2] = other.z != id ? 0.f : ds[4 * w + 2];
            ds[4 * w + 3] = other.w != id ? 0.f : ds[4 * w + 3];
          }
        if (scoring.prefixed || !docs)
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = 8 * (r >> 2) + (r & 3) >= limit - at ? 0.f : ds[r];
      }
      if constexpr (kHalf<T>) keep_in_range<false, ND>(ds, dq, raise);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Frag<T> f = result_frag<T>(ds, w);
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[n] = mma<T>(Lds::down(kt, 32 * u + 16 * w, n, la), f, dq[n]);
      }
    }
  };
  if (first < last) fetch(kt0, vt0);
  for (int tile = first; tile < last; tile += 2) {
    step(tile, kt0, vt0, kt1, vt1);
    if (tile + 1 < last) step(tile + 1, kt1, vt1, kt0, vt0);
  }
  if (!real) return;
  lower<T, ND>(dq, raise);
  if (a.splits > 1)
    write_gradient<float, ND>(a.part + ((int64_t)blockIdx.y * a.n * a.hq * a.lq + stat) * D, dq, 1.0f, D, lane);
  else
    write_gradient<T, ND>(static_cast<T*>(a.dq) + b * a.dqb + h * a.dqh + (int64_t)i * a.dql, dq, ds_scale<CAP>(a),
                          a.d, lane);
}

template <typename T, int D>
constexpr int dkv_waves() {
  return D * sizeof(T) >= 256 ? 1 : D * sizeof(T) == 64 ? 4 : 2;
}

// dk and dv: 128 keys of a key head, the query tiles of its heads streaming.
template <typename T, int D, Cap CAP>
__global__ __launch_bounds__(kThreads, (dkv_waves<T, D>())) void attention_dkv_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  typedef Tile<T, D> Lds;
  __shared__ __attribute__((aligned(16))) char qt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char gt0[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char qt1[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) char gt1[kTile * Lds::kRow];
  __shared__ __attribute__((aligned(16))) float stats0[2 * kTile];  // lse, -delta
  __shared__ __attribute__((aligned(16))) float stats1[2 * kTile];
  __shared__ unsigned odd[2][2];  // of dout, of q
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.lk + kOwn - 1) / kOwn;
  const bool docs = a.qdoc.ids != nullptr;
  int item, block;
  Part part;
  place(blockIdx.x, a.n * a.hk, blocks, docs ? 2 : 1, item, block, part.part);  // a prefix: the first have most rows
  const int b = item / a.hk, hk = item % a.hk;
  if (part.part == 1 && !is_mixed(a.kdoc, b, block)) return;
  const int j0 = block * kOwn;
  const int j = j0 + 32 * wave + (lane & 31);
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const int* ids = docs ? a.qdoc.ids + (int64_t)b * a.qdoc.stride : nullptr;
  const int* own_ids = docs ? a.kdoc.ids + (int64_t)b * a.kdoc.stride : nullptr;
  part.first_id = docs ? own_ids[j0] : 0;
  const int own = docs && j < a.lk ? own_ids[j] : 0;
  const bool real = j < a.lk && (!docs || part.has(own));  // keys of the other part are left to it
  const int id = own < 0 || !real ? -2 : own;  // -2 matches no row
  const int off = a.lk - a.lq;
  const T* k = static_cast<const T*>(a.k) + b * a.kb + hk * a.kh + (int64_t)j * a.kl;
  const T* v = static_cast<const T*>(a.v) + b * a.vb + hk * a.vh + (int64_t)j * a.vl;

  Frag<T> kf[NK], vf[NK];
#pragma unroll
  for (int s = 0; s < NK; ++s) {
    kf[s] = frag_global(k, s, a.d, lane, real);
    vf[s] = frag_global(v, s, a.d, lane, real);
  }
  f16v dk[ND], dv[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) dk[n] = dv[n] = f16v(0.f);

  const Meeting meet = meeting<kWaves>(wave, j0, a.lk, [&](int row) { return query_tiles(a, b, row, prefix, &part); });
  const int first = meet.all.x, last = meet.all.y;
  const int tiles = last - first;
  const int2 mine = split_steps(tiles * a.group, blockIdx.y, a.splits);
  typedef Stream<T, D, kTile, kThreads> Load;
  Rows<T, kTile> qrows, grows;
  int h = hk * a.group + (tiles > 0 ? mine.x / tiles : 0), tile = first + (tiles > 0 ? mine.x % tiles : 0) - 1;
  int fetched = h, at_tile = tile + 1;  // head and tile of the next fetch
  bool begun = false;
  auto fetch = [&](char* qt, char* gt, float* stats) {
    if (at_tile == first || !begun) {
      begun = true;
      qrows.begin(static_cast<const T*>(a.q) + b * a.qb + fetched * a.qh, a.ql, at_tile * kTile, a.lq, a.d);
      grows.begin(static_cast<const T*>(a.dout) + b * a.gb + fetched * a.gh, a.gl, at_tile * kTile, a.lq, a.d);
    }
    Load::load(qt, qrows, t);
    Load::load(gt, grows, t);
    qrows.next();
    grows.next();
    const int64_t row = ((int64_t)b * a.hq + fetched) * a.lq;
    if (wave < 2) load_floats(stats + wave * kTile, (wave == 0 ? a.lse : a.delta) + row, at_tile * kTile, a.lq, lane);
    if (++at_tile == last) {
      at_tile = first;
      ++fetched;
    }
  };
  Scoring scoring = scoring_of(a, hk * a.group);
  float raise = kDsRaise<T>;
  // One tile, while the next one is on its way into the other arrays.
  auto step = [&](bool more, char* qt, char* gt, float* stats, char* next_qt, char* next_gt, float* next_stats) {
    if (++tile == last) {
      tile = first;
      ++h;
    }
    const int i0 = tile * kTile;
    const bool partial = meet.partial(tile);
    if (a.slopes) scoring.slope = a.slopes[h];
    arrive();
    if (more) fetch(next_qt, next_gt, next_stats);
    if (partial) {
      if (t < 4) odd[t >> 1][t & 1] = 0u;
      __syncthreads();
      Load::clean(qt, odd[1], t);
      Load::clean(gt, odd[0], t);
      __syncthreads();
    }
    if (meet.skips(tile)) return;
    const int la = fresh<D == 128>(lane);
    const bool masked = meet.masked(tile);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f16v s = f16v(0.f), ds;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f4 delta = *reinterpret_cast<const f4*>(stats + kTile + 32 * u + 8 * w + 4 * half);
#pragma unroll
        for (int r = 0; r < 4; ++r) ds[4 * w + r] = delta[r];
      }
      // With one or two waves a SIMD little else covers the latency of the reads: they are issued a group ahead of
      // their products, the first operands of the gradients before the scores are worked on.  (Left to itself the
      // compiler reads one operand, waits for it and multiplies: 710 us for 624 of 2 x 16 heads of 4096 rows of 128.)
      constexpr bool kAhead = sizeof(T) == 2 && D >= 64;
      Frag<T> along[2][NK], down[2][ND][2];
      auto read_along = [&](int n) {
        along[0][n] = Lds::along(qt, 32 * u, n, la);
        along[1][n] = Lds::along(gt, 32 * u, n, la);
      };
      auto read_down = [&](int w) {
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          down[0][n][w] = Lds::down(gt, 32 * u + 16 * w, n, la);
          down[1][n][w] = Lds::down(qt, 32 * u + 16 * w, n, la);
        }
      };
      if constexpr (kAhead) {
#pragma unroll
        for (int n = 0; n < NK / 2; ++n) read_along(n);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        if constexpr (kAhead) {
          if (n == 0) {
#pragma unroll
            for (int e = NK / 2; e < NK; ++e) read_along(e);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (n == NK / 2) {
            __builtin_amdgcn_sched_barrier(0);
            read_down(0);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
          read_along(n);
        }
        s = mma<T>(along[0][n], kf[n], s);
        ds = mma<T>(along[1][n], vf[n], ds);
      }
      const int at = i0 + 32 * u + 4 * half;
      const float c = scores<T, CAP>(scoring, s, ds, at, j - off);
      const float raised = kHalf<T> ? __builtin_ldexpf(1.0f, (int)(raise - kRaise)) : 1.0f;  // p is raised already
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f4 lse = *reinterpret_cast<const f4*>(stats + 32 * u + 8 * w + 4 * half);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[4 * w + r] = __builtin_amdgcn_exp2f(fmaf(s[4 * w + r], c, kHalf<T> ? kRaise - lse[r] : -lse[r]));
          ds[4 * w + r] *= s[4 * w + r];
          if constexpr (kHalf<T>) ds[4 * w + r] *= raised;
        }
      }
      if (masked) {
        auto hide = [&](int r, bool so) {
          s[r] = so ? 0.f : s[r];
          ds[r] = so ? 0.f : ds[r];
        };
        if (docs)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int4 other = *reinterpret_cast<const int4*>(ids + i0 + 32 * u + 4 * half + 8 * w);
            hide(4 * w, other.x != id);
            hide(4 * w + 1, other.y != id);
            hide(4 * w + 2, other.z != id);
            hide(4 * w + 3, other.w != id);
          }
        if (i0 + kTile > a.lq)  // rows past the end, whose zeros give a p that may be infinite
#pragma unroll
          for (int r = 0; r < 16; ++r) hide(r, 8 * (r >> 2) + (r & 3) >= a.lq - at);
        if (scoring.prefixed && j >= prefix)  // else every row sees the key
#pragma unroll
          for (int r = 0; r < 16; ++r) hide(r, 8 * (r >> 2) + (r & 3) < j - off - at);
      }
      if constexpr (kHalf<T>) keep_in_range<D == 128, ND>(ds, dk, raise);
      if constexpr (kAhead) {
        read_down(1);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Frag<T> p = result_frag<T>(s, w), f = result_frag<T>(ds, w);
        if constexpr (!kAhead) read_down(w);
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          dv[n] = mma<T>(down[0][n][w], p, dv[n]);
          dk[n] = mma<T>(down[1][n][w], f, dk[n]);
        }
      }
      if (partial && odd[0][u]) {
        // Values of dout that were zeroed in LDS, for the keys that their rows see.
        const int odd_half = fresh<true>(lane) >> 5;  // else the offsets below stay in registers over the loop
        const T* gh = static_cast<const T*>(a.dout) + b * a.gb + h * a.gh;
        for (int r = 0; r < 32; ++r) {
          if (((odd[0][u] >> r) & 1u) == 0u) continue;
          const int i = i0 + 32 * u + r;
          if (j >= limit_of(a, i, prefix) || (docs && ids[i] != id)) continue;
          const T* row = gh + (int64_t)i * a.gl;
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const Vec<float, 4> value = load_as_float<T, 4>(row + min(32 * n + 8 * w + 4 * odd_half, a.d - 4));
#pragma unroll
              for (int e = 0; e < 4; ++e) dv[n][4 * w + e] += fabsf(value[e]) < INFINITY ? 0.f : value[e];
            }
        }
      }
    }
  };
  if (mine.x < mine.y) fetch(qt0, gt0, stats0);
  for (int s = mine.x; s < mine.y; s += 2) {
    step(s + 1 < mine.y, qt0, gt0, stats0, qt1, gt1, stats1);
    if (s + 1 < mine.y) step(s + 2 < mine.y, qt1, gt1, stats1, qt0, gt0, stats0);
  }
  if (!real) return;
  lower<T, ND>(dk, raise);
  lower<T, ND>(dv, kRaise);
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.n * a.hk * a.lk;
    float* part = a.part + (2 * blockIdx.y * rows + ((int64_t)b * a.hk + hk) * a.lk + j) * D;
    if (a.dk) write_gradient<float, ND>(part, dk, 1.0f, D, lane);
    if (a.dv) write_gradient<float, ND>(part + rows * D, dv, 1.0f, D, lane);
    return;
  }
  if (a.dk)
    write_gradient<T, ND>(static_cast<T*>(a.dk) + b * a.dkb + hk * a.dkh + (int64_t)j * a.dkl, dk, ds_scale<CAP>(a),
                          a.d, lane);
  if (a.dv)
    write_gradient<T, ND>(static_cast<T*>(a.dv) + b * a.dvb + hk * a.dvh + (int64_t)j * a.dvl, dv, 1.0f, a.d, lane);
}

// Adds the parts of gradients in order: four values a thread.  blockIdx.y: which of up to two gradients.
struct SumArgs {
  const float* part;  // (splits, gradients, rows, D)
  void* out[2];       // null: left out
  int64_t sb[2], sh[2], sl[2];
  float scale[2];
  int rows, heads, length, d, splits, gradients;
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_sum_kernel(SumArgs a) {
  const int which = blockIdx.y;
  const int at = blockIdx.x * kThreads + threadIdx.x, row = at / (D / 4), e = at % (D / 4) * 4;
  if (row >= a.rows || e >= a.d || !a.out[which]) return;
  const float* part = a.part + ((int64_t)which * a.rows + row) * D + e;
  f4 sum = *reinterpret_cast<const f4*>(part);
#pragma unroll 4
  for (int s = 1; s < a.splits; ++s) sum += *reinterpret_cast<const f4*>(part + (int64_t)s * a.gradients * a.rows * D);
  const int i = row % a.length, bh = row / a.length;
  T* out = static_cast<T*>(a.out[which]) + bh / a.heads * a.sb[which] + bh % a.heads * a.sh[which] + i * a.sl[which];
  Vec<float, 4> v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = sum[r] * a.scale[which];
  store_rounded<T, 4>(out + e, v);
}

// Parts of each block's stream where the blocks alone do not fill the chip: as many workgroups as it holds at a time
// (one a CU where a row has 256 bytes or more, else two), of at least `least` steps.  From the shape only, so that a
// shape's sums have one order.  2000 rows of 16 heads on 4 key heads of 128, bf16: 183 us, 382 in one part; 1500 rows
// of 8 heads on 2 of 64: 74, 174 in one part; 256 rows of 2 x 16 heads of 32, whose 64 blocks have 4 steps each: 24 as
// one part, 30 as two.
constexpr int kMostParts = 64;
int part_count(int64_t blocks, int64_t steps, int elem, int head_dim) {
  const int64_t slots = padded(head_dim) * elem_bytes(elem) >= 256 ? 256 : 512;
  const int64_t least = elem != CTMR_ELEM_F32 ? 4 : padded(head_dim) >= 64 ? 1 : 2;
  return (int)std::max<int64_t>(1, std::min<int64_t>({slots / blocks, steps / least, kMostParts}));
}
int query_parts(const ctmr_masked_attention_desc* d) {
  return part_count((int64_t)d->n * d->q_heads * ceil_div(d->lq, kOwn), ceil_div(d->lk, kTile), d->elem, d->head_dim);
}
int key_parts(const ctmr_masked_attention_desc* d) {
  return part_count((int64_t)d->n * d->k_heads * ceil_div(d->lk, kOwn),
                    ceil_div(d->lq, kTile) * (d->q_heads / d->k_heads), d->elem, d->head_dim);
}

// Bytes of delta in the workspace; the parts follow, dq's and then, in the same place, dk's and dv's.
int64_t delta_bytes(const ctmr_masked_attention_desc* d) {
  return ceil_div((int64_t)d->n * d->q_heads * d->lq * 4, 16) * 16;
}

template <typename T, int D, Cap CAP>
int launch(Args a, int qparts, int kparts, hipStream_t st) {
  const unsigned parts = a.qdoc.ids ? 2u : 1u;
  a.splits = a.dq ? qparts : 1;
  const unsigned q_blocks = a.n * a.hq * (unsigned)ceil_div(a.lq, kOwn) * parts;
  hipLaunchKernelGGL((attention_dq_kernel<T, D, CAP>), dim3(q_blocks, a.splits), dim3(kThreads), 0, st, a);
  int rc = check_launch("attention_dq");
  if (rc) return rc;
  if (a.splits > 1) {
    SumArgs s = {a.part, {a.dq, nullptr}, {a.dqb, 0}, {a.dqh, 0}, {a.dql, 0}, {ds_scale<CAP>(a), 0.f},
                 a.n * a.hq * a.lq, a.hq, a.lq, a.d, a.splits, 1};
    hipLaunchKernelGGL((attention_sum_kernel<T, D>), dim3((unsigned)ceil_div((int64_t)s.rows * (D / 4), kThreads)),
                       dim3(kThreads), 0, st, s);
    rc = check_launch("attention_sum");
    if (rc) return rc;
  }
  if (!a.dk && !a.dv) return rc;
  a.splits = kparts;
  const unsigned k_blocks = a.n * a.hk * (unsigned)ceil_div(a.lk, kOwn) * parts;
  hipLaunchKernelGGL((attention_dkv_kernel<T, D, CAP>), dim3(k_blocks, a.splits), dim3(kThreads), 0, st, a);
  rc = check_launch("attention_dkv");
  if (rc || a.splits == 1) return rc;
  SumArgs s = {a.part, {a.dk, a.dv}, {a.dkb, a.dvb}, {a.dkh, a.dvh}, {a.dkl, a.dvl}, {ds_scale<CAP>(a), 1.0f},
               a.n * a.hk * a.lk, a.hk, a.lk, a.d, a.splits, 2};
  hipLaunchKernelGGL((attention_sum_kernel<T, D>), dim3((unsigned)ceil_div((int64_t)s.rows * (D / 4), kThreads), 2),
                     dim3(kThreads), 0, st, s);
  return check_launch("attention_sum");
}

}  // namespace
}  // namespace attn
}  // namespace ctmr

using namespace ctmr;
using namespace ctmr::attn;

extern "C" {

int64_t ctmr_masked_attention_backward_workspace_bytes(const ctmr_masked_attention_desc* d) {
  const int rc = check_desc(d);
  if (rc) return rc;
  const int64_t q = query_parts(d), k = key_parts(d);
  const int64_t qbytes = q > 1 ? q * d->n * d->q_heads * d->lq * padded(d->head_dim) * 4 : 0;
  const int64_t kbytes = k > 1 ? 2 * k * d->n * d->k_heads * d->lk * padded(d->head_dim) * 4 : 0;
  return delta_bytes(d) + std::max(qbytes, kbytes);
}

int ctmr_masked_attention_backward(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v,
                                   const float* slopes, const int32_t* prefixes, const void* plan, const void* out,
                                   const void* rest, const float* lse, const void* dout, const int64_t* dout_strides,
                                   void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                                   const int64_t* dv_strides, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t need = ctmr_masked_attention_backward_workspace_bytes(d);
  if (need < 0) return (int)need;
  if (!q || !k || !v || !out || !lse || !dout || !dout_strides || (dq && !dq_strides) || (dk && !dk_strides) ||
      (dv && !dv_strides))
    return fail(CTMR_E_INVALID, "null pointer");
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest | (uintptr_t)dout |
        (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)plan) & 15) != 0)
    return fail(CTMR_E_INVALID, "tensors and the document plan must start on 16-byte boundaries");
  for (const int64_t* s : {dout_strides, d->out_strides}) {
    const int rc = check_strides(d, s, d->lq);
    if (rc) return rc;
  }
  for (const int64_t* s : {dq ? dq_strides : nullptr, dk ? dk_strides : nullptr, dv ? dv_strides : nullptr})
    if (s && (s[0] | s[1] | s[2]) % 4 != 0)
      return fail(CTMR_E_INVALID, "strides of the gradients must be multiples of 4 values");
  if ((int64_t)workspace_bytes < need || !workspace || ((uintptr_t)workspace & 15) != 0) {
    set_error("attention workspace: %zu bytes given, %lld needed on a 16-byte boundary", workspace_bytes,
              (long long)need);
    return CTMR_E_WORKSPACE;
  }
  if (!dq && !dk && !dv) return CTMR_OK;
  Args a = make_args(d, q, k, v, slopes, prefixes, plan);
  a.out = const_cast<void*>(out), a.rest = const_cast<void*>(rest), a.lse = const_cast<float*>(lse), a.dout = dout;
  a.dq = dq, a.dk = dk, a.dv = dv, a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + delta_bytes(d));
  a.ob = d->out_strides[0], a.oh = d->out_strides[1], a.ol = d->out_strides[2];
  a.gb = dout_strides[0], a.gh = dout_strides[1], a.gl = row_stride(dout_strides, d->lq, d->head_dim);
  if (dq) a.dqb = dq_strides[0], a.dqh = dq_strides[1], a.dql = dq_strides[2];
  if (dk) a.dkb = dk_strides[0], a.dkh = dk_strides[1], a.dkl = dk_strides[2];
  if (dv) a.dvb = dv_strides[0], a.dvh = dv_strides[1], a.dvl = dv_strides[2];
  const int qparts = query_parts(d), kparts = key_parts(d);
  hipStream_t st = (hipStream_t)stream;
  const bool cap = d->softcap > 0.f;
#define CTMR_ATTENTION_CASE(T, D)                                             \
  if (!cap) return launch<T, D, kNoCap>(a, qparts, kparts, st);               \
  if constexpr (sizeof(T) == 2)                                               \
    if (shifted_cap<T>(d->softcap)) return launch<T, D, kShiftedCap>(a, qparts, kparts, st); \
  return launch<T, D, kExactCap>(a, qparts, kparts, st);
#define CTMR_ATTENTION_TYPE(T)              \
  switch (padded(d->head_dim)) {            \
    case 32: CTMR_ATTENTION_CASE(T, 32)     \
    case 64: CTMR_ATTENTION_CASE(T, 64)     \
    default: CTMR_ATTENTION_CASE(T, 128)    \
  }
  if (d->elem == CTMR_ELEM_F32) CTMR_ATTENTION_TYPE(float)
  if (d->elem == CTMR_ELEM_BF16) CTMR_ATTENTION_TYPE(__bf16)
  CTMR_ATTENTION_TYPE(_Float16)
#undef CTMR_ATTENTION_TYPE
#undef CTMR_ATTENTION_CASE
}

}  // extern "C"
