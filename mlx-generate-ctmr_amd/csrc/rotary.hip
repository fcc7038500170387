// Rotary positions of up to four axes (depth, height, width, ...) for the heads
// of q and k, in one launch.
//
// The first sum(width_a) values of a head are split into a section per axis;
// pair i of section a (values i and i + width_a / 2 of it) turns by
//   angle = position_a * base^(-2 i / width_a)
//   (p, q) -> (p cos - q sin, p sin + q cos)
// and the rest of the head passes as it is.  The gradient is the turn by -angle.
//
// Angles are position * (base^.. / 2 pi) in fp64, reduced to a part of a turn
// before they are rounded to fp32: at a position of 10^5 an fp32 product would be
// off by 10^-2.  Bound by HBM (each value read and written once, 16 bytes a
// thread); a workgroup computes the sines of its tokens once, in LDS, for all
// heads.  2 x 30011 tokens of 32 + 8 heads of 128, bf16: 272 us, 4.5 TB/s, where a copy
// of that size reaches 4.7.
#include "elements.hpp"

#include <algorithm>

namespace ctmr {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 1024;  // pairs of a workgroup's table: tokens x pairs

struct RotaryArgs {
  const void* in[2];
  void* out[2];
  int64_t in_b[2], in_h[2], in_l[2];     // strides in values; the last is 1
  int64_t out_b[2], out_h[2], out_l[2];
  int heads[2];
  const void* positions;
  int64_t pos_b;                          // values between batch items, 0 for shared positions
  int n, l, d, axes, pairs, tokens;       // tokens: of a workgroup
  int start[4], half[4];                  // pair slots: first of a section, pairs in it
  float way;                              // +1, or -1 for the gradient
  double turns[CTMR_ROTARY_MAX_PAIRS];    // of a pair at position 1
};

// POS: 0 int32, 1 int64, 2 fp32 positions.
template <typename T, int V, int POS>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 table[kTable];
  const int b = blockIdx.y;
  const int l0 = blockIdx.x * a.tokens, count = min(a.tokens, a.l - l0);
  for (int i = threadIdx.x; i < count * a.pairs; i += kThreads) {
    const int t = i / a.pairs, p = i % a.pairs;
    int axis = 0;
#pragma unroll
    for (int s = 1; s < 4; ++s)
      if (s < a.axes && p >= a.start[s]) axis = s;
    const int64_t at = (int64_t)b * a.pos_b + (int64_t)(l0 + t) * a.axes + axis;
    double pos;
    if constexpr (POS == 0) pos = (double)static_cast<const int*>(a.positions)[at];
    else if constexpr (POS == 1) pos = (double)static_cast<const int64_t*>(a.positions)[at];
    else pos = (double)static_cast<const float*>(a.positions)[at];
    const double turn = pos * a.turns[p];
    float sine, cosine;
    sincospif(2.0f * (float)(turn - rint(turn)), &sine, &cosine);
    table[i] = float2{cosine, a.way * sine};
  }
  __syncthreads();
  // Items: V pairs, or V pairs of the values that pass, of a head of a token.
  const int slots = a.d / (2 * V), turned = a.pairs / V;
  const int heads = a.heads[0] + a.heads[1];
  const int items = count * heads * slots;
  for (int i = threadIdx.x; i < items; i += kThreads) {
    const int slot = i % slots, rest = i / slots;
    const int head = rest % heads, t = rest / heads;
    const int which = head >= a.heads[0] ? 1 : 0;
    const int h = head - (which ? a.heads[0] : 0);
    const int p = slot * V;
    const T* in = static_cast<const T*>(a.in[which]) + b * a.in_b[which] + h * a.in_h[which] +
                  (int64_t)(l0 + t) * a.in_l[which];
    T* out = static_cast<T*>(a.out[which]) + b * a.out_b[which] + h * a.out_h[which] +
             (int64_t)(l0 + t) * a.out_l[which];
    if (slot >= turned) {
      const int at = 2 * p;  // two vectors side by side, as they are
      const Vec<T, V> u = *reinterpret_cast<const Vec<T, V>*>(in + at);
      const Vec<T, V> w = *reinterpret_cast<const Vec<T, V>*>(in + at + V);
      *reinterpret_cast<Vec<T, V>*>(out + at) = u;
      *reinterpret_cast<Vec<T, V>*>(out + at + V) = w;
      continue;
    }
    int start = 0, half = a.half[0];
#pragma unroll
    for (int s = 1; s < 4; ++s)
      if (s < a.axes && p >= a.start[s]) {
        start = a.start[s];
        half = a.half[s];
      }
    const int at = start + p;  // 2 * start + (p - start)
    const Vec<float, V> u = load_as_float<T, V>(in + at), w = load_as_float<T, V>(in + at + half);
    Vec<float, V> x, y;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float2 cs = table[t * a.pairs + p + k];
      x[k] = u[k] * cs.x - w[k] * cs.y;
      y[k] = u[k] * cs.y + w[k] * cs.x;
    }
    store_rounded<T, V>(out + at, x);
    store_rounded<T, V>(out + at + half, y);
  }
}

template <typename T, int V>
void launch(const RotaryArgs& a, int pos, dim3 grid, hipStream_t st) {
  if (pos == CTMR_POS_I32) hipLaunchKernelGGL((rotary_kernel<T, V, 0>), grid, dim3(kThreads), 0, st, a);
  else if (pos == CTMR_POS_I64) hipLaunchKernelGGL((rotary_kernel<T, V, 1>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((rotary_kernel<T, V, 2>), grid, dim3(kThreads), 0, st, a);
}

}  // namespace
}  // namespace ctmr

using namespace ctmr;

extern "C" int ctmr_rotary(const ctmr_rotary_desc* d, const void* q, const void* k, const void* positions,
                           const double* turns, void* q_out, void* k_out, void* stream) {
  if (!d) return fail(CTMR_E_INVALID, "null descriptor");
  if (d->n <= 0 || d->l <= 0 || d->head_dim <= 0 || d->q_heads <= 0 || d->k_heads < 0)
    return fail(CTMR_E_INVALID, "non-positive dimension");
  if (!valid_elem(d->elem) || d->position_type < CTMR_POS_I32 || d->position_type > CTMR_POS_F32)
    return fail(CTMR_E_INVALID, "bad element type");
  if (d->axes < 1 || d->axes > 4) return fail(CTMR_E_INVALID, "one to four axes");
  if (!q || !q_out || !positions || !turns || (d->k_heads > 0 && (!k || !k_out)))
    return fail(CTMR_E_INVALID, "null pointer");
  if (d->head_dim % 2 != 0) return fail(CTMR_E_INVALID, "head_dim must be even");
  if (d->n > 65535 || d->head_dim > 2 * CTMR_ROTARY_MAX_PAIRS || (int64_t)d->q_heads + d->k_heads > (1 << 15))
    return fail(CTMR_E_UNSUPPORTED, "too many batch items, heads or values a head");
  RotaryArgs a = {};
  const int bytes = elem_bytes(d->elem);
  int64_t sum = 0;
  int width = 16 / bytes;  // values a vector: divides every section's half and the rest's
  auto fit = [&](int64_t v) {
    while (width > 1 && v % width != 0) width >>= 1;
  };
  for (int s = 0; s < d->axes; ++s) {
    if (d->widths[s] <= 0 || d->widths[s] % 2 != 0) return fail(CTMR_E_INVALID, "sections have positive even widths");
    a.start[s] = (int)(sum / 2);
    a.half[s] = d->widths[s] / 2;
    sum += d->widths[s];
    if (sum > d->head_dim) return fail(CTMR_E_INVALID, "sections are wider than the head");
    fit(a.half[s]);
  }
  fit((d->head_dim - sum) / 2);
  const int tensors = d->k_heads > 0 ? 2 : 1;
  for (int t = 0; t < tensors; ++t) {
    a.in[t] = t ? k : q;
    a.out[t] = t ? k_out : q_out;
    a.heads[t] = t ? d->k_heads : d->q_heads;
    const int64_t* in = t ? d->k_strides : d->q_strides;
    const int64_t* out = t ? d->k_out_strides : d->q_out_strides;
    a.in_b[t] = in[0], a.in_h[t] = in[1], a.in_l[t] = in[2];
    a.out_b[t] = out[0], a.out_h[t] = out[1], a.out_l[t] = out[2];
    for (int i = 0; i < 3; ++i) {
      fit(in[i]);
      fit(out[i]);
    }
    while (width > 1 && (((uintptr_t)a.in[t] | (uintptr_t)a.out[t]) % (uintptr_t)(width * bytes)) != 0) width >>= 1;
  }
  a.positions = positions;
  a.pos_b = d->position_batch_stride;
  a.n = d->n, a.l = d->l, a.d = d->head_dim, a.axes = d->axes, a.pairs = (int)(sum / 2);
  a.way = d->inverse ? -1.0f : 1.0f;
  std::copy(turns, turns + a.pairs, a.turns);
  // Tokens of a workgroup: as many as the table holds, fewer while there would be under 2048 workgroups.
  int tokens = std::max(1, std::min(16, kTable / a.pairs));
  while (tokens > 1 && ceil_div(a.l, tokens) * a.n < 2048) tokens >>= 1;
  a.tokens = tokens;
  if (ceil_div(a.l, tokens) > (1 << 23)) return fail(CTMR_E_UNSUPPORTED, "too many tokens");  // 2^32 threads
  const dim3 grid((unsigned)ceil_div(a.l, tokens), a.n);
  hipStream_t st = (hipStream_t)stream;
#define CTMR_ROTARY_CASE(T, W) \
  case W:                      \
    launch<T, W>(a, d->position_type, grid, st); \
    break;
  if (d->elem == CTMR_ELEM_F32) switch (width) {
      CTMR_ROTARY_CASE(float, 4) CTMR_ROTARY_CASE(float, 2) CTMR_ROTARY_CASE(float, 1)
    }
  else if (d->elem == CTMR_ELEM_BF16) switch (width) {
      CTMR_ROTARY_CASE(__bf16, 8) CTMR_ROTARY_CASE(__bf16, 4) CTMR_ROTARY_CASE(__bf16, 2) CTMR_ROTARY_CASE(__bf16, 1)
    }
  else switch (width) {
      CTMR_ROTARY_CASE(_Float16, 8) CTMR_ROTARY_CASE(_Float16, 4) CTMR_ROTARY_CASE(_Float16, 2)
      CTMR_ROTARY_CASE(_Float16, 1)
    }
#undef CTMR_ROTARY_CASE
  return check_launch("rotary");
}
