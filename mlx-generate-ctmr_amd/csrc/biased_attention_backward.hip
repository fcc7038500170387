// Gradients of the masked attention with a position bias, the table's among them.  The
// kernels are those of masked_attention_backward.hpp with the bias looked up, each type's
// compiled in a source of its own (biased_gradients_*.hip); the table's gradient comes from
// the workgroups' sums by distance.
#include "masked_attention_backward.hpp"

namespace ctmr {
namespace attn {
namespace {

// One workgroup a head: the sums of all items and workgroups for each distance, a quarter of them a thread, then those
// of each row of the table, all in one order and in fp64.
__global__ __launch_bounds__(1024) void table_gradient_kernel(const float* part, const int* rows, int items, int hq, int slots,
                                                              int table_rows, int elem, void* out) {
  __shared__ double sums[4][kDistances];
  __shared__ int row_of[kDistances];
  const int h = blockIdx.x, number = threadIdx.x & (kDistances - 1), quarter = threadIdx.x / kDistances;
  double sum = 0.0;
  for (int b = 0; b < items; ++b) {
    const float* from = part + ((int64_t)b * hq + h) * slots * kDistances + number;
#pragma unroll 8
    for (int s = quarter; s < slots; s += 4) sum += (double)from[(int64_t)s * kDistances];
  }
  sums[quarter][number] = sum;
  if (quarter == 0) row_of[number] = rows[number];
  __syncthreads();
  if (quarter == 0) sums[0][number] = (sums[0][number] + sums[1][number]) + (sums[2][number] + sums[3][number]);
  __syncthreads();
  // Eight threads a row, a distance each in turn.
  const int lane = threadIdx.x & 7;
  for (int row = threadIdx.x >> 3; row < table_rows; row += 128) {
    double total = 0.0;
#pragma unroll 4
    for (int n = lane; n < kDistances; n += 8) total += row_of[n] == row ? sums[0][n] : 0.0;
#pragma unroll
    for (int m = 4; m > 0; m >>= 1) total += __shfl_xor(total, m);
    if (lane == 0) store_param(out, elem, (int64_t)row * hq + h, (float)total);
  }
}

int slots_of(const ctmr_masked_attention_desc* d, bool documents) {
  return query_parts(d) * (documents ? 2 : 1) * (int)ceil_div(d->lq, kOwn);
}

int64_t table_bytes(const ctmr_masked_attention_desc* d, bool documents) {
  return (int64_t)d->n * d->q_heads * slots_of(d, documents) * kDistances * 4;
}

}  // namespace
}  // namespace attn
}  // namespace ctmr

using namespace ctmr;
using namespace ctmr::attn;

extern "C" {

int64_t ctmr_biased_attention_backward_workspace_bytes(const ctmr_masked_attention_desc* d, int32_t documents) {
  const int64_t bytes = ctmr_masked_attention_backward_workspace_bytes(d);
  return bytes < 0 ? bytes : round_up(bytes, 16) + table_bytes(d, documents != 0);
}

int ctmr_biased_attention_backward(const ctmr_masked_attention_desc* d, const ctmr_buckets_desc* buckets, const void* q,
                                   const void* k, const void* v, const float* slopes, const int32_t* prefixes,
                                   const void* plan, const void* bucket_plan, const void* table, const void* out,
                                   const void* rest, const float* lse, const void* dout, const int64_t* dout_strides,
                                   void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                                   const int64_t* dv_strides, void* dtable, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const int64_t need = ctmr_biased_attention_backward_workspace_bytes(d, plan != nullptr);
  if (need < 0) return (int)need;
  Args a;
  int rc = check_gradients(d, q, k, v, slopes, prefixes, plan, out, rest, lse, dout, dout_strides, dq, dq_strides, dk,
                           dk_strides, dv, dv_strides, workspace, workspace_bytes, need, a);
  if (!rc) rc = check_buckets(d, buckets);
  if (rc) return rc;
  if (!bucket_plan || !table || ((uintptr_t)bucket_plan & 15) != 0)
    return fail(CTMR_E_INVALID, "a bias needs its table and a plan of places on a 16-byte boundary");
  if (!dq && !dk && !dv && !dtable) return CTMR_OK;
  Bias bias = make_bias(d, buckets, bucket_plan, table);
  bias.slots = slots_of(d, plan != nullptr);
  if (dtable)
    bias.part = (float*)((char*)workspace + round_up(ctmr_masked_attention_backward_workspace_bytes(d), 16));
  hipStream_t st = (hipStream_t)stream;
  const auto run = d->elem == CTMR_ELEM_F32    ? run_biased_gradients<float>
                   : d->elem == CTMR_ELEM_BF16 ? run_biased_gradients<__bf16>
                                               : run_biased_gradients<_Float16>;
  rc = run(a, bias, bias_steps(buckets), query_parts(d), key_parts(d), st);
  if (rc || !dtable) return rc;
  hipLaunchKernelGGL(table_gradient_kernel, dim3(d->q_heads), dim3(1024), 0, st, bias.part, bias.rows, d->n, d->q_heads,
                     bias.slots, buckets->table_rows, buckets->table_elem, dtable);
  return check_launch("table_gradient");
}

}  // extern "C"
