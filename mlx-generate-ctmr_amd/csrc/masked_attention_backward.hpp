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
// 4096 rows, every key, bf16, both kernels: heads of 32 330 us, of 64 501 (686 TFLOP/s
// of the five products, 960 of the seven), of 128 997; fp16 383, 581, 1160 (the powers of
// two below: two operations a score in dk and dv, half a one in dq); fp32, 2 x 8 heads of
// 2048 rows of 32: 251 (120 of the seven, where a library product of 8192^3 reaches 153).
// With a position bias on 16x16x16 and its table's gradient (position_bias.hpp): bf16, heads
// of 32 655 us, of 64 815, of 128 1858, for a table of 16 bits 605, 761, 1800, and for one
// without a gradient 498, 650, 1621; fp32 as above on 16x16x8 318, 276 without.  dk and dv spill
// scalar registers there (117 to 196 of the bias' arguments, 65 to 75 without a bias), and with
// heads of 32 and 16 bits 26 to 64 vector registers.
//
// fp16's range is far smaller than what ds spans, so every row of dq and every key of
// dk (a lane's column) has a power of two of its own that ds is multiplied by: the sums
// start with 2^40 and move down, like a running maximum, when a ds passes 2^15.  Values
// of ds down to 2^-38 of the largest that the row or key has met count, whatever other
// rows, heads and documents hold.  p is raised by 2^15.  All comes out of the sums again
// at the end, exactly.
#pragma once

#include "position_bias.hpp"

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
// compiler computes and selects.)  `add` adds to the capped scores.
template <Cap CAP>
__device__ __forceinline__ float units_of(const Scoring& a) {
  return CAP == kNoCap ? a.scale * kLog2e : a.cap * (kLog2e * kCapUnits<CAP>);
}
template <typename T, Cap CAP, typename F>
__device__ __forceinline__ float scores(const Scoring& a, f16v& s, f16v& ds, int at, int x, F add) {
  const float c = units_of<CAP>(a);
  if constexpr (CAP != kNoCap) {
    cap_scores<CAP>(s, a.scale / a.cap);
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= cap_slope<CAP>(s[r]);
  }
  add(s);
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

// Adds to the gradient of r what a 32 x 32 block of scores' gradients gives, in two parts or three.
template <int ST>
__device__ __forceinline__ void add_row_gradient(f16v (&dr)[HotTile<ST>::kBlocks], f16v ds, bool third, const char* hot,
                                                 int row, int lane) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    if (p == 2 && !third) break;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Frag<__bf16> f = result_frag<__bf16>(ds, w);
#pragma unroll
      for (int n = 0; n < HotTile<ST>::kBlocks; ++n)
        dr[n] = mma<__bf16>(HotTile<ST>::down(hot, row + 16 * w, n, lane), f, dr[n]);
#pragma unroll
      for (int e = 0; e < 8; ++e) ds[8 * w + e] -= (float)f[e];
    }
  }
}

// A workgroup's gradients of r, added over its rows by distance: thread t's is distance t.  A wave's 32 rows at a time
// go through LDS (32 rows of the columns, their pieces of four turned by the row).
template <int ST>
__device__ __forceinline__ void add_distances(const Bias& bias, const f16v (&dr)[HotTile<ST>::kBlocks], unsigned places,
                                              bool real, float* lds, float* out, int t) {
  constexpr int kWidth = 32 * HotTile<ST>::kBlocks;
  const auto turned = [](int piece, int row) { return piece ^ (row & (ST == 6 && piece >= 16 ? 7 : 15)); };
  __shared__ unsigned row_places[32];
  const int lane = t & 63, half = lane >> 5, wave = t >> 6, own = lane & 31;
  int axis = 0;  // of distance t; the last axis has the numbers that no distance has, too
  while (axis + 1 < bias.axes && t >= bias.first_number[axis + 1]) ++axis;
  const int extent = bias.extents[axis], distance = t - bias.first_number[axis] - (extent - 1);
  float sum = 0.f;
  for (int w = 0; w < kWaves; ++w) {
    __syncthreads();
    if (wave == w) {
      if (half == 0) row_places[own] = places;
#pragma unroll
      for (int n = 0; n < HotTile<ST>::kBlocks; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f4 v = {0.f, 0.f, 0.f, 0.f};
          if (real) v = f4{dr[n][4 * q], dr[n][4 * q + 1], dr[n][4 * q + 2], dr[n][4 * q + 3]};
          *reinterpret_cast<f4*>(lds + own * kWidth + 4 * turned(8 * n + 2 * q + half, own)) = v;
        }
    }
    __syncthreads();
    for (int i = 0; i < 32; ++i) {
      const int x = (int)((row_places[i] >> (8 * axis)) & 255) + distance;
      if (x < 0 || x >= extent) continue;
      const int column = bias.first_column[axis] + x;
      sum += lds[i * kWidth + 4 * turned(column >> 2, i) + (column & 3)];
    }
  }
  out[t] = sum;
}

// Waves a SIMD that the registers are kept for.  16-bit, 2 x 16 heads of 4096 rows, both kernels: heads of 32 with four
// 330 us (a few registers spill), with three 351; heads of 64 with three for dk and dv too (20 spill) 577 us, with two
// there 501.  With a bias dq has up to 64 more sums a lane: heads of 32 with 96 columns, 8192 rows on 32x32x8, both kernels
// with two 1182 us, with three 1514 (ds in two parts).
template <typename T, int D, int ST>
constexpr int dq_waves() {
  if (ST > 0) return D * sizeof(T) >= 256 ? 1 : 2;
  return D * sizeof(T) >= 512 ? 1 : D * sizeof(T) == 64 ? 4 : D * sizeof(T) == 128 ? 3 : 2;
}

extern __shared__ __attribute__((aligned(16))) char bias_values[];  // of a position bias (lay_out_bias)

// dq and delta: 128 query rows of a head, key tiles streaming.
template <typename T, int D, Cap CAP, int ST>
__global__ __launch_bounds__(kThreads, (dq_waves<T, D, ST>())) void attention_dq_kernel(Args a, BiasOf<ST> bias) {
  constexpr int NK = D / 16, ND = D / 32;
  typedef Tile<T, D> Lds;
  constexpr bool kOneHot = one_hot<T, D, ST>();
  __shared__ __attribute__((aligned(16))) char hot0[HotTile<ST>::kBytes];
  __shared__ __attribute__((aligned(16))) char hot1[kOneHot ? 16 : HotTile<ST>::kBytes];
  __shared__ __attribute__((aligned(16))) unsigned words0[kTile];
  __shared__ __attribute__((aligned(16))) unsigned words1[kTile];
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
  float* table_part = nullptr;
  if constexpr (ST > 0) {
    const int64_t slot = ((int64_t)blockIdx.y * (docs ? 2 : 1) + part.part) * blocks + block;
    if (bias.part) table_part = bias.part + (((int64_t)b * a.hq + h) * bias.slots + slot) * kDistances;
  }
  if (part.part == 1 && !is_mixed(a.qdoc, b, block)) {
    if (table_part) table_part[t] = 0.f;
    return;
  }
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

  // The matrix units round sums of 16-bit products to one side, so each dr (and with 16-bit heads each ds) has a bias that
  // the table's sums over rows and keys add up, the more the longer they are: of the table's gradient 2.5e-6 at 4096 rows with
  // 16-bit heads, 8e-7 with fp32 ones and 1.4e-6 at 16384.  Odd rows have g and all that is made of it with the other
  // sign, and it cancels (below 2e-7 of a drift from 256 to 16384 rows, heads of 32 and 128).
  constexpr bool kFlips = ST > 0;
  const float flip = kFlips && (lane & 1) ? -1.f : 1.f;
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
      const int64_t at = b * a.ob + h * a.oh + (int64_t)i * a.ol;
      if (ST > 0 && a.rest) {  // fp32
        const Frag<float> rf = frag_global(static_cast<const float*>(a.rest) + at, s, a.d, lane, real);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[s][e], rf[e], delta);
      } else if (a.rest) {
        const Frag<T> rf = frag_global(static_cast<const T*>(a.rest) + at, s, a.d, lane, real);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[s][e], (float)rf[e], delta);
      }
    }
  }
  delta = half_sum(delta);
  if (real && half == 0 && blockIdx.y == 0) a.delta[stat] = -delta;
  if (!a.dq && !table_part) return;
  if constexpr (kFlips) {
    delta *= flip;
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      if constexpr (sizeof(T) == 2)
        gf[s] = __builtin_bit_cast(Frag<T>, __builtin_bit_cast(u4, gf[s]) ^ (lane & 1 ? 0x80008000u : 0u));
      else
        gf[s] *= flip;
    }
  }
  const float lse = real ? a.lse[stat] : INFINITY;
  float raise = kDsRaise<T>;
  f16v dq[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) dq[n] = f16v(0.f);
  unsigned places = 0u;
  unsigned word = 0u;
  f16v dr[HotTile<ST>::kBlocks];  // of r
  if constexpr (ST > 0) {
    if (real) places = bias.query_places[b * bias.query_item + i];
    word = row_word<kSingle<T, D>>(bias, b, i, a.lq);
    lay_out_bias<kSingle<T, D>, kThreads>(bias, bias_values, h, a.hq, kLog2e / units_of<CAP>(scoring),
                                          t);  // arrive() comes before its use
#pragma unroll
    for (int n = 0; n < HotTile<ST>::kBlocks; ++n) dr[n] = f16v(0.f);
  }

  const Meeting meet = meeting<kWaves>(wave, i0, a.lq, [&](int row) { return key_tiles(a, b, row, prefix, &part); });
  const int2 mine = split_steps(meet.all.y - meet.all.x, blockIdx.y, a.splits);
  const int first = meet.all.x + mine.x, last = meet.all.x + mine.y;
  Rows<T, kTile> krows, vrows;
  krows.begin(k, a.kl, first * kTile, a.lk, a.d);
  vrows.begin(v, a.vl, first * kTile, a.lk, a.d);
  typedef Stream<T, D, kTile, kThreads> Load;
  auto fetch_hot = [&](int tile, char* hot) {
    if constexpr (ST > 0)
      HotTile<ST>::template load<kThreads>(hot, bias.key_hot + b * bias.hot_item * HotTile<ST>::kRow, tile * kTile, a.lk, t);
  };
  auto fetch = [&](int tile, char* kt, char* vt, char* hot, unsigned* words) {
    Load::load(kt, krows, t);
    Load::load(vt, vrows, t);
    if constexpr (ST > 0) {
      if (!kOneHot && table_part) fetch_hot(tile, hot);
      if (wave == 0) load_words(words, (kSingle<T, D> ? bias.key_places : bias.key_codes) + b * bias.key_item, tile * kTile, a.lk, lane);
    }
    krows.next();
    vrows.next();
  };
  // One tile, while the next one is on its way into the other pair of arrays.
  auto step = [&](int tile, char* kt, char* vt, char* hot, unsigned* words, char* next_kt, char* next_vt, char* next_hot,
                  unsigned* next_words) {
    const int k0 = tile * kTile;
    const bool partial = meet.partial(tile);
    arrive();
    if constexpr (ST > 0 && kOneHot)
      if (table_part) {
        fetch_hot(tile, hot);
        arrive();
      }
    if (tile + 1 < last) fetch(tile + 1, next_kt, next_vt, next_hot, next_words);
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
      if constexpr (ST > 0 && CAP == kNoCap)  // the products are added to the bias
        apply_bias<kSingle<T, D>, true, false, kBiasRows<D>>(s, bias_values, word, words + 32 * u, la);
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        s = mma<T>(Lds::along(kt, 32 * u, n, la), qf[n], s);
        ds = mma<T>(Lds::along(vt, 32 * u, n, la), gf[n], ds);
      }
      const int at = k0 + 32 * u + 4 * half;
      f16v db = ds;  // of the bias: before the cap's slope
      const float c = scores<T, CAP>(scoring, s, ds, at, pos, [&](f16v& s) {
        if constexpr (ST > 0 && CAP != kNoCap)
          apply_bias<kSingle<T, D>, true, true, kBiasRows<D>>(s, bias_values, word, words + 32 * u, la);
      });
      if constexpr (ST > 0 && CAP != kNoCap) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, kHalf<T> ? raise - lse : -lse));
          ds[r] *= p;
          db[r] *= p;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] *= __builtin_amdgcn_exp2f(fmaf(s[r], c, kHalf<T> ? raise - lse : -lse));
      }
      // (As a function of ds or db this kept ds in memory: heads of 32 with a cap past 256 spilled 112 registers, 9 so.)
      if (masked) {
#pragma unroll
        for (int which = 0; which < (ST > 0 && CAP != kNoCap ? 2 : 1); ++which) {
          f16v& hidden = which == 0 ? ds : db;
          // a visible key whose values were zeroed in LDS because they are not finite: no gradient is
          const unsigned set = partial ? odd[u] >> (4 * half) : 0u;
          if (set)
#pragma unroll
            for (int r = 0; r < 16; ++r) hidden[r] = (set >> (8 * (r >> 2) + (r & 3))) & 1u ? NAN : hidden[r];
          if (docs)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int4 other = *reinterpret_cast<const int4*>(ids + k0 + 32 * u + 4 * half + 8 * w);
              hidden[4 * w] = other.x != id ? 0.f : hidden[4 * w];
              hidden[4 * w + 1] = other.y != id ? 0.f : hidden[4 * w + 1];
              hidden[4 * w + 2] = other.z != id ? 0.f : hidden[4 * w + 2];
              hidden[4 * w + 3] = other.w != id ? 0.f : hidden[4 * w + 3];
            }
          if (scoring.prefixed || !docs)
#pragma unroll
            for (int r = 0; r < 16; ++r) hidden[r] = 8 * (r >> 2) + (r & 3) >= limit - at ? 0.f : hidden[r];
        }
      }
      const float raised = raise;  // of db
      if constexpr (kHalf<T>) keep_in_range<false, ND>(ds, dq, raise);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Frag<T> f = result_frag<T>(ds, w);
#pragma unroll
        for (int n = 0; n < ND; ++n) dq[n] = mma<T>(Lds::down(kt, 32 * u + 16 * w, n, la), f, dq[n]);
      }
      if constexpr (ST > 0)
        if (table_part) {
          if constexpr (CAP == kNoCap) db = ds;
          if constexpr (kHalf<T>) db *= __builtin_ldexpf(1.0f, -(int)(CAP == kNoCap ? raise : raised));
          add_row_gradient<ST>(dr, db, sizeof(T) == 4 || wide_table(bias), hot, 32 * u, la);
        }
    }
  };
  char* const other = kOneHot ? hot0 : hot1;
  if (first < last) fetch(first, kt0, vt0, hot0, words0);
  for (int tile = first; tile < last; tile += 2) {
    step(tile, kt0, vt0, hot0, words0, kt1, vt1, other, words1);
    if (tile + 1 < last) step(tile + 1, kt1, vt1, other, words1, kt0, vt0, hot0, words0);
  }
  if constexpr (kFlips) {
#pragma unroll
    for (int n = 0; n < ND; ++n) dq[n] *= flip;
#pragma unroll
    for (int n = 0; n < HotTile<ST>::kBlocks; ++n) dr[n] *= flip;
  }
  if constexpr (ST > 0) {
    if (table_part) add_distances<ST>(bias, dr, places, real, reinterpret_cast<float*>(hot0), table_part, t);
    if (!a.dq) return;
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
template <typename T, int D, Cap CAP, int ST>
__global__ __launch_bounds__(kThreads, (dkv_waves<T, D>())) void attention_dkv_kernel(Args a, BiasOf<ST> bias) {
  constexpr int NK = D / 16, ND = D / 32;
  typedef Tile<T, D> Lds;
  __shared__ __attribute__((aligned(16))) unsigned words0[kTile];
  __shared__ __attribute__((aligned(16))) unsigned words1[kTile];
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
  unsigned word = 0u;
  if constexpr (ST > 0) {
    word = key_word<kSingle<T, D>>(bias, b, j, a.lk) - (kSingle<T, D> ? bias.reach : 0u);
  }
  const int query_room = (a.lq + kTile - 1) / kTile * kTile;  // words past the last row are a row's, too
  auto fetch = [&](char* qt, char* gt, float* stats, unsigned* words) {
    if (at_tile == first || !begun) {
      begun = true;
      qrows.begin(static_cast<const T*>(a.q) + b * a.qb + fetched * a.qh, a.ql, at_tile * kTile, a.lq, a.d);
      grows.begin(static_cast<const T*>(a.dout) + b * a.gb + fetched * a.gh, a.gl, at_tile * kTile, a.lq, a.d);
    }
    Load::load(qt, qrows, t);
    Load::load(gt, grows, t);
    if constexpr (ST > 0)
      if (wave == 2) load_words(words, (kSingle<T, D> ? bias.query_places : bias.query_codes) + b * bias.query_item, at_tile * kTile,
                   query_room, lane);
    qrows.next();
    grows.next();
    const int64_t row = ((int64_t)b * a.hq + fetched) * a.lq;
    if (wave < 2) load_words(stats + wave * kTile, (wave == 0 ? a.lse : a.delta) + row, at_tile * kTile, a.lq, lane);
    if (++at_tile == last) {
      at_tile = first;
      ++fetched;
    }
  };
  Scoring scoring = scoring_of(a, hk * a.group);
  float raise = kDsRaise<T>;
  // One tile, while the next one is on its way into the other arrays.
  auto step = [&](bool more, char* qt, char* gt, float* stats, unsigned* words, char* next_qt, char* next_gt,
                  float* next_stats, unsigned* next_words) {
    if (++tile == last) {
      tile = first;
      ++h;
    }
    const int i0 = tile * kTile;
    const bool partial = meet.partial(tile);
    if (a.slopes) scoring.slope = a.slopes[h];
    arrive();
    if (more) fetch(next_qt, next_gt, next_stats, next_words);
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
      if constexpr (ST > 0 && CAP == kNoCap)  // the products are added to the bias
        apply_bias<kSingle<T, D>, false, false, kBiasRows<D>>(s, bias_values, word, words + 32 * u, la);
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
      const float c = scores<T, CAP>(scoring, s, ds, at, j - off, [&](f16v& s) {
        if constexpr (ST > 0 && CAP != kNoCap)
          apply_bias<kSingle<T, D>, false, true, kBiasRows<D>>(s, bias_values, word, words + 32 * u, la);
      });
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
  if (mine.x < mine.y) fetch(qt0, gt0, stats0, words0);
  int head = -1;  // whose bias LDS holds
  auto turn = [&]() {
    if constexpr (ST > 0) {
      const int next = h + (tile + 1 == last ? 1 : 0);  // of the next step
      if (next == head) return;
      head = next;
      __syncthreads();  // the last head's is read; arrive() comes before the next one's use
      lay_out_bias<kSingle<T, D>, kThreads>(bias, bias_values, head, a.hq, kLog2e / units_of<CAP>(scoring), t);
    }
  };
  for (int s = mine.x; s < mine.y; s += 2) {
    turn();
    step(s + 1 < mine.y, qt0, gt0, stats0, words0, qt1, gt1, stats1, words1);
    if (s + 1 < mine.y) {
      turn();
      step(s + 2 < mine.y, qt1, gt1, stats1, words1, qt0, gt0, stats0, words0);
    }
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

template <typename T, int D, Cap CAP, int ST>
int launch(Args a, const BiasOf<ST>& bias, int qparts, int kparts, hipStream_t st) {
  const unsigned parts = a.qdoc.ids ? 2u : 1u, bytes = bias_bytes<T, D>(bias);
  bool table = false;
  if constexpr (ST > 0) table = bias.part != nullptr;
  a.splits = a.dq || table ? qparts : 1;
  const unsigned q_blocks = a.n * a.hq * (unsigned)ceil_div(a.lq, kOwn) * parts;
  hipLaunchKernelGGL((attention_dq_kernel<T, D, CAP, ST>), dim3(q_blocks, a.splits), dim3(kThreads), bytes, st, a,
                     bias);
  int rc = check_launch("attention_dq");
  if (rc) return rc;
  if (a.splits > 1 && a.dq) {
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
  constexpr int kAny = ST > 0 ? kBias : 0;
  if constexpr (ST > 0)
    hipLaunchKernelGGL((attention_dkv_kernel<T, D, CAP, kAny>), dim3(k_blocks, a.splits), dim3(kThreads), bytes, st, a,
                       BiasOf<kAny>{bias});
  else
    hipLaunchKernelGGL((attention_dkv_kernel<T, D, CAP, 0>), dim3(k_blocks, a.splits), dim3(kThreads), 0, st, a, bias);
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
