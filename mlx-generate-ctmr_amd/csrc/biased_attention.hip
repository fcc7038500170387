// Masked attention with a position bias: the entry point of its forward call.  The
// kernels are those of masked_attention_forward.hpp with the bias looked up.
#include "masked_attention_forward.hpp"

using namespace ctmr;
using namespace ctmr::attn;

extern "C" int ctmr_biased_attention(const ctmr_masked_attention_desc* d, const ctmr_buckets_desc* buckets, const void* q,
                                     const void* k, const void* v, const float* slopes, const int32_t* prefixes,
                                     const void* plan, const void* bucket_plan, const void* table, int32_t fine,
                                     void* out, void* rest, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const int64_t need = ctmr_masked_attention_workspace_bytes(d);
  if (need < 0) return (int)need;
  int rc = check_call(d, q, k, v, plan, out, rest, workspace, workspace_bytes, need);
  if (!rc) rc = check_buckets(d, buckets);
  if (rc) return rc;
  if (!bucket_plan || !table || ((uintptr_t)bucket_plan & 15) != 0)
    return fail(CTMR_E_INVALID, "a bias needs its table and a plan of places on a 16-byte boundary");
  Args a = make_args(d, q, k, v, slopes, prefixes, plan);
  a.out = out, a.rest = rest, a.wide_rest = 1, a.lse = lse, a.part = (float*)workspace, a.splits = split_count(d);
  a.ob = d->out_strides[0], a.oh = d->out_strides[1], a.ol = d->out_strides[2];
  const Bias bias = make_bias(d, buckets, bucket_plan, table);
  const bool few = few_rows(d);
  hipStream_t st = (hipStream_t)stream;
  auto run = [&](auto type, auto width) {
    typedef decltype(type) T;
    constexpr int D = decltype(width)::value;
    if constexpr (sizeof(T) == 2)
      if (fine) {
        if constexpr (std::is_same_v<T, __bf16>)
          if (bias.elem == CTMR_ELEM_F32) return launch<T, D>(a, BiasOf<kFinestBias>{bias}, few, st);
        return launch<T, D>(a, BiasOf<kFineBias>{bias}, few, st);
      }
    return launch<T, D>(a, BiasOf<kBias>{bias}, few, st);
  };
  auto of_type = [&](auto type) {
    switch (padded(d->head_dim)) {
      case 32: return run(type, std::integral_constant<int, 32>());
      case 64: return run(type, std::integral_constant<int, 64>());
      default: return run(type, std::integral_constant<int, 128>());
    }
  };
  if (d->elem == CTMR_ELEM_F32) return of_type(0.0f);
  return d->elem == CTMR_ELEM_BF16 ? of_type((__bf16)0.0f) : of_type((_Float16)0.0f);
}
