// The entry points of the masked attention's gradients.  The kernels are in
// masked_attention_backward.hpp.
#include "masked_attention_backward.hpp"

namespace ctmr {
namespace attn {

// Bytes of delta in the workspace; the parts follow, dq's and then, in the same place, dk's and dv's.
int64_t delta_bytes(const ctmr_masked_attention_desc* d) {
  return ceil_div((int64_t)d->n * d->q_heads * d->lq * 4, 16) * 16;
}

int check_gradients(const ctmr_masked_attention_desc* d, const void* q, const void* k, const void* v, const float* slopes,
                    const int32_t* prefixes, const void* plan, const void* out, const void* rest, const float* lse,
                    const void* dout, const int64_t* dout_strides, void* dq, const int64_t* dq_strides, void* dk,
                    const int64_t* dk_strides, void* dv, const int64_t* dv_strides, void* workspace,
                    size_t workspace_bytes, int64_t need, Args& a) {
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
  a = make_args(d, q, k, v, slopes, prefixes, plan);
  a.out = const_cast<void*>(out), a.rest = const_cast<void*>(rest), a.lse = const_cast<float*>(lse), a.dout = dout;
  a.dq = dq, a.dk = dk, a.dv = dv, a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + delta_bytes(d));
  a.ob = d->out_strides[0], a.oh = d->out_strides[1], a.ol = d->out_strides[2];
  a.gb = dout_strides[0], a.gh = dout_strides[1], a.gl = row_stride(dout_strides, d->lq, d->head_dim);
  if (dq) a.dqb = dq_strides[0], a.dqh = dq_strides[1], a.dql = dq_strides[2];
  if (dk) a.dkb = dk_strides[0], a.dkh = dk_strides[1], a.dkl = dk_strides[2];
  if (dv) a.dvb = dv_strides[0], a.dvh = dv_strides[1], a.dvl = dv_strides[2];
  return CTMR_OK;
}

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
  Args a;
  const int rc = check_gradients(d, q, k, v, slopes, prefixes, plan, out, rest, lse, dout, dout_strides, dq, dq_strides, dk,
                                 dk_strides, dv, dv_strides, workspace, workspace_bytes, need, a);
  if (rc) return rc;
  if (!dq && !dk && !dv) return CTMR_OK;
  const int qparts = query_parts(d), kparts = key_parts(d);
  hipStream_t st = (hipStream_t)stream;
  const bool cap = d->softcap > 0.f;
  const BiasOf<0> none;
#define CTMR_ATTENTION_CASE(T, D)                                             \
  if (!cap) return launch<T, D, kNoCap>(a, none, qparts, kparts, st);         \
  if constexpr (sizeof(T) == 2)                                               \
    if (shifted_cap<T>(d->softcap)) return launch<T, D, kShiftedCap>(a, none, qparts, kparts, st); \
  return launch<T, D, kExactCap>(a, none, qparts, kparts, st);
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
