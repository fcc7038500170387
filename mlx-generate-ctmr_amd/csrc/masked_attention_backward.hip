// Gradients of the masked attention (masked_attention.hip), for fp32 and bf16.
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
// products for the five of the formulas (scores and g . v twice), but no atomics:
// each sum has one order, and the gradients are bit-identical run to run.  p and ds
// are rounded to the operands' type for their products, half a step of it on each
// term of an fp32 sum.
//
// fp16 is refused: without a scale that follows the data ds leaves its range.
#include "masked_attention.hpp"

#include <algorithm>
#include <cmath>

namespace ctmr {
namespace attn {
namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kOwn = 32 * kWaves;  // rows that a workgroup keeps in registers

// Products of a 32 x 32 block -> log2 scores in units of 1 / c (c returned) and, with a cap, 1 - t^2 in `slope_of`.
// Row r of a lane is `at` + 8 (r / 4) + r % 4; `x` is where the distance to it is zero.
template <typename T>
__device__ __forceinline__ float scores(const Args& a, f16v& s, f16v& slope_of, int at, int x, float slope) {
  float c = a.scale * kLog2e;
  if (a.cap > 0.f) {
    const float in = a.scale / a.cap, out = a.cap * kLog2e;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float t = tanh_of<T>(s[r] * in);
      s[r] = out * t;
      slope_of[r] = fmaf(-t, t, 1.0f);
    }
    c = 1.0f;
  }
  if (a.slopes) {
    const float per = slope * kLog2e;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fmaf(-per, fabsf((float)(at + 8 * (r >> 2) + (r & 3) - x)), s[r] * c);
    c = 1.0f;
  }
  return c;
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

// dq and delta: 128 query rows of a head, key tiles streaming.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, D == 128 ? 1 : 2) void attention_dq_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  constexpr int KS = tile_stride<T, D>(BOTH), VS = tile_stride<T, D>(ALONG);
  __shared__ __attribute__((aligned(16))) T kt[kTile * KS];
  __shared__ __attribute__((aligned(16))) T vt[kTile * VS];
  __shared__ __attribute__((aligned(16))) int key_ids[kTile];
  __shared__ unsigned odd[2];
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.lq + kOwn - 1) / kOwn;
  int item, block;
  place(blockIdx.x, a.n * a.hq, blocks, item, block);
  if (a.prefixed) block = blocks - 1 - block;
  const int b = item / a.hq, h = item % a.hq;
  const int i0 = block * kOwn;
  const int i = i0 + 32 * wave + (lane & 31);
  const bool real = i < a.lq;
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const bool docs = a.qdoc.ids != nullptr;
  const int* ids = docs ? a.kdoc.ids + (int64_t)b * a.kdoc.stride : nullptr;
  const int limit = real ? limit_of(a, i, prefix) : 0, id = docs && real ? row_id(a, b, i) : -2;
  const int pos = i + a.lk - a.lq;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
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
  if (real && half == 0) a.delta[stat] = delta;
  if (!a.dq) return;
  const float lse = real ? a.lse[stat] : INFINITY;
  f16v dq[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) dq[n] = f16v(0.f);

  const Meeting meet = meeting<kWaves>(wave, i0, a.lq, [&](int row) { return key_tiles(a, b, row, prefix); });
  const int first = meet.all.x, last = meet.all.y;
  Stream<T, D, kTile, kThreads> ks, vs;
  int other_id = 0;
  auto fetch = [&](int tile) {
    ks.fetch(k, a.kl, tile * kTile, a.lk, a.d, t);
    vs.fetch(v, a.vl, tile * kTile, a.lk, a.d, t);
    if (docs && t < kTile) other_id = ids[tile * kTile + t];
  };
  if (first < last) fetch(first);
  for (int tile = first; tile < last; ++tile) {
    const int k0 = tile * kTile;
    const bool partial = meet.partial(tile);
    __syncthreads();  // the last tile is read
    if (t < 2) odd[t] = 0u;
    if (docs && t < kTile) key_ids[t] = other_id;
    if (partial) {
      __syncthreads();
      ks.template store<true>(kt, KS, odd, t);
    } else {
      ks.template store<false>(kt, KS, nullptr, t);
    }
    vs.template store<false>(vt, VS, nullptr, t);
    __syncthreads();
    if (tile + 1 < last) fetch(tile + 1);
    if (meet.skips(tile)) continue;
    const bool masked = meet.masked(tile) || (partial && (odd[0] | odd[1]) != 0u);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f16v s = f16v(0.f), ds = f16v(0.f), slope_of = f16v(1.f);
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        s = mma<T>(frag_along(kt, KS, 32 * u, n, lane), qf[n], s);
        ds = mma<T>(frag_along(vt, VS, 32 * u, n, lane), gf[n], ds);
      }
      const int at = k0 + 32 * u + 4 * half;
      const float c = scores<T>(a, s, slope_of, at, pos, slope);
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (ds[r] - delta);
      if (a.cap > 0.f) ds *= slope_of;
      if (masked) {
        const unsigned set = odd[u];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          int4 other = {id, id, id, id};
          if (docs) other = *reinterpret_cast<const int4*>(key_ids + 32 * u + 4 * half + 8 * w);
          const int key_id[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // a visible key whose values were zeroed in LDS because they are not finite: no gradient is
            if ((set >> (8 * w + 4 * half + r)) & 1u) ds[4 * w + r] = NAN;
            if (at + 8 * w + r >= limit || key_id[r] != id) ds[4 * w + r] = 0.f;
          }
        }
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Frag<T> f = result_frag<T>(ds, w);
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[n] = mma<T>(frag_down(kt, KS, 32 * u + 16 * w, n, lane), f, dq[n]);
      }
    }
  }
  if (real)
    write_gradient<T, ND>(static_cast<T*>(a.dq) + b * a.dqb + h * a.dqh + (int64_t)i * a.dql, dq, a.scale, a.d, lane);
}

// dk and dv: 128 keys of a key head, the query tiles of its heads streaming.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, D == 128 ? 1 : 2) void attention_dkv_kernel(Args a) {
  constexpr int NK = D / 16, ND = D / 32;
  constexpr int S = tile_stride<T, D>(BOTH);
  __shared__ __attribute__((aligned(16))) T qt[kTile * S];
  __shared__ __attribute__((aligned(16))) T gt[kTile * S];
  __shared__ __attribute__((aligned(16))) float stats[2][kTile];  // lse, delta
  __shared__ __attribute__((aligned(16))) int query_ids[kTile];
  __shared__ unsigned odd[2][2];  // of dout, of q
  const int t = threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (a.lk + kOwn - 1) / kOwn;
  int item, block;
  place(blockIdx.x, a.n * a.hk, blocks, item, block);  // with a prefix the first keys have the most rows
  const int b = item / a.hk, hk = item % a.hk;
  const int j0 = block * kOwn;
  const int j = j0 + 32 * wave + (lane & 31);
  const bool real = j < a.lk;
  const int prefix = a.prefixed ? prefix_of(a, b) : 0;
  const bool docs = a.qdoc.ids != nullptr;
  const int* ids = docs ? a.qdoc.ids + (int64_t)b * a.qdoc.stride : nullptr;
  // padding keys match no row: rows' negative ids are -1
  const int own_id = docs && real ? a.kdoc.ids[(int64_t)b * a.kdoc.stride + j] : 0;
  const int id = own_id < 0 ? -2 : own_id;
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

  const Meeting meet = meeting<kWaves>(wave, j0, a.lk, [&](int row) { return query_tiles(a, b, row, prefix); });
  const int first = meet.all.x, last = meet.all.y;
  const int tiles = last - first, steps = tiles * a.group;
  Stream<T, D, kTile, kThreads> qs, gs;
  float stat = 0.f;
  int other_id = 0;
  auto fetch = [&](int step) {
    const int h = hk * a.group + step / tiles, tile = first + step % tiles;
    qs.fetch(static_cast<const T*>(a.q) + b * a.qb + h * a.qh, a.ql, tile * kTile, a.lq, a.d, t);
    gs.fetch(static_cast<const T*>(a.dout) + b * a.gb + h * a.gh, a.gl, tile * kTile, a.lq, a.d, t);
    const int i = tile * kTile + (t & (kTile - 1));
    if (t < 2 * kTile) {
      const float* from = t < kTile ? a.lse : a.delta;
      stat = i < a.lq ? from[((int64_t)b * a.hq + h) * a.lq + i] : t < kTile ? INFINITY : 0.f;
      if (docs) other_id = ids[i];
    }
  };
  if (steps > 0) fetch(0);
  for (int step = 0; step < steps; ++step) {
    const int h = hk * a.group + step / tiles, tile = first + step % tiles, i0 = tile * kTile;
    const bool partial = meet.partial(tile);
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    __syncthreads();
    if (t < 4) odd[t >> 1][t & 1] = 0u;
    if (t < 2 * kTile) stats[t / kTile][t % kTile] = stat;
    if (docs && t < kTile) query_ids[t] = other_id;
    if (partial) {
      __syncthreads();
      qs.template store<true>(qt, S, odd[1], t);
      gs.template store<true>(gt, S, odd[0], t);
    } else {
      qs.template store<false>(qt, S, nullptr, t);
      gs.template store<false>(gt, S, nullptr, t);
    }
    __syncthreads();
    if (step + 1 < steps) fetch(step + 1);
    if (meet.skips(tile)) continue;
    const bool masked = meet.masked(tile);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f16v s = f16v(0.f), ds = f16v(0.f), slope_of = f16v(1.f);
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        s = mma<T>(frag_along(qt, S, 32 * u, n, lane), kf[n], s);
        ds = mma<T>(frag_along(gt, S, 32 * u, n, lane), vf[n], ds);
      }
      const int at = i0 + 32 * u + 4 * half;
      const float c = scores<T>(a, s, slope_of, at, j - off, slope);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f4 lse = *reinterpret_cast<const f4*>(&stats[0][32 * u + 8 * w + 4 * half]);
        const f4 delta = *reinterpret_cast<const f4*>(&stats[1][32 * u + 8 * w + 4 * half]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[4 * w + r] = __builtin_amdgcn_exp2f(fmaf(s[4 * w + r], c, -lse[r]));
          ds[4 * w + r] = s[4 * w + r] * (ds[4 * w + r] - delta[r]);
        }
      }
      if (a.cap > 0.f) ds *= slope_of;
      unsigned hidden = 0u;
      if (masked) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          int4 other = {id, id, id, id};
          if (docs) other = *reinterpret_cast<const int4*>(query_ids + 32 * u + 4 * half + 8 * w);
          const int query_id[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (j >= limit_of(a, at + 8 * w + r, prefix) || query_id[r] != id) {
              s[4 * w + r] = ds[4 * w + r] = 0.f;
              hidden |= 1u << (4 * w + r);
            }
        }
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Frag<T> p = result_frag<T>(s, w), f = result_frag<T>(ds, w);
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          dv[n] = mma<T>(frag_down(gt, S, 32 * u + 16 * w, n, lane), p, dv[n]);
          dk[n] = mma<T>(frag_down(qt, S, 32 * u + 16 * w, n, lane), f, dk[n]);
        }
      }
      if (partial && odd[0][u]) {
        // Values of dout that were zeroed in LDS, for the keys that their rows see.  A lane knows 16 of the 32
        // rows; the other half of the wave, which has the same keys, knows the rest.
        const unsigned others = (unsigned)__shfl_xor((int)hidden, 32);
        const T* gh = static_cast<const T*>(a.dout) + b * a.gb + h * a.gh;
        for (int r = 0; r < 32; ++r) {
          if (((odd[0][u] >> r) & 1u) == 0u) continue;
          const int bit = 4 * (r >> 3) + (r & 3);
          const unsigned seen_by = ((r >> 2) & 1) == half ? hidden : others;
          if (((seen_by >> bit) & 1u) != 0u) continue;
          const T* row = gh + (int64_t)(i0 + 32 * u + r) * a.gl;
#pragma unroll
          for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const Vec<float, 4> value = load_as_float<T, 4>(row + min(32 * n + 8 * w + 4 * half, a.d - 4));
#pragma unroll
              for (int e = 0; e < 4; ++e) dv[n][4 * w + e] += fabsf(value[e]) < INFINITY ? 0.f : value[e];
            }
        }
      }
    }
  }
  if (!real) return;
  if (a.dk)
    write_gradient<T, ND>(static_cast<T*>(a.dk) + b * a.dkb + hk * a.dkh + (int64_t)j * a.dkl, dk, a.scale, a.d, lane);
  if (a.dv)
    write_gradient<T, ND>(static_cast<T*>(a.dv) + b * a.dvb + hk * a.dvh + (int64_t)j * a.dvl, dv, 1.0f, a.d, lane);
}

template <typename T, int D>
int launch(const Args& a, hipStream_t st) {
  hipLaunchKernelGGL((attention_dq_kernel<T, D>), dim3(a.n * a.hq * (unsigned)ceil_div(a.lq, kOwn)), dim3(kThreads), 0,
                     st, a);
  const int rc = check_launch("attention_dq");
  if (rc || (!a.dk && !a.dv)) return rc;
  hipLaunchKernelGGL((attention_dkv_kernel<T, D>), dim3(a.n * a.hk * (unsigned)ceil_div(a.lk, kOwn)), dim3(kThreads),
                     0, st, a);
  return check_launch("attention_dkv");
}

}  // namespace
}  // namespace attn
}  // namespace ctmr

using namespace ctmr;
using namespace ctmr::attn;

extern "C" {

int64_t ctmr_masked_attention_backward_workspace_bytes(const ctmr_masked_attention_desc* d) {
  const int rc = check_desc(d);
  return rc ? rc : (int64_t)d->n * d->q_heads * d->lq * 4;
}

int ctmr_masked_attention_backward(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v,
                                   const float* slopes, const int32_t* prefixes, const void* plan, const void* out,
                                   const void* rest, const float* lse, const void* dout, const int64_t* dout_strides, void* dq,
                                   const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                                   const int64_t* dv_strides, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t need = ctmr_masked_attention_backward_workspace_bytes(d);
  if (need < 0) return (int)need;
  if (d->elem == CTMR_ELEM_F16) return fail(CTMR_E_UNSUPPORTED, "attention has no fp16 gradient");
  if (!q || !k || !v || !out || !lse || !dout || !dout_strides || (dq && !dq_strides) || (dk && !dk_strides) ||
      (dv && !dv_strides))
    return fail(CTMR_E_INVALID, "null pointer");
  if ((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)rest | (uintptr_t)dout | (uintptr_t)dq |
        (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)plan) & 15) != 0)
    return fail(CTMR_E_INVALID, "tensors and the document plan must start on 16-byte boundaries");
  const int bytes = elem_bytes(d->elem);
  for (const int64_t* s : {dout_strides, d->out_strides}) {
    if (s[0] < 0 || s[1] < 0 || s[2] < 0 || (s[0] | s[1] | s[2]) * bytes % 16 != 0)
      return fail(CTMR_E_INVALID, "strides must be multiples of 16 bytes and not negative");
    if (s[2] * bytes > (1ll << 31) / kTile - 4096) return fail(CTMR_E_UNSUPPORTED, "row stride too large");
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
  a.ob = d->out_strides[0], a.oh = d->out_strides[1], a.ol = d->out_strides[2];
  a.gb = dout_strides[0], a.gh = dout_strides[1], a.gl = dout_strides[2];
  if (dq) a.dqb = dq_strides[0], a.dqh = dq_strides[1], a.dql = dq_strides[2];
  if (dk) a.dkb = dk_strides[0], a.dkh = dk_strides[1], a.dkl = dk_strides[2];
  if (dv) a.dvb = dv_strides[0], a.dvh = dv_strides[1], a.dvl = dv_strides[2];
  hipStream_t st = (hipStream_t)stream;
#define CTMR_ATTENTION_CASE(T)              \
  switch (padded(d->head_dim)) {            \
    case 32: return launch<T, 32>(a, st);   \
    case 64: return launch<T, 64>(a, st);   \
    default: return launch<T, 128>(a, st);  \
  }
  if (d->elem == CTMR_ELEM_F32) CTMR_ATTENTION_CASE(float)
  CTMR_ATTENTION_CASE(__bf16)
#undef CTMR_ATTENTION_CASE
}

}  // extern "C"
