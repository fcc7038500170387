// The gradients' kernels of the masked attention with a position bias for one type of
// heads, which the including source instantiates.
#pragma once

#include "masked_attention_backward.hpp"

namespace ctmr {
namespace attn {
namespace {

template <typename T, int D, int NE>
int run_width(const Args& a, const BiasOf<NE>& bias, int qparts, int kparts, hipStream_t st) {
  if (a.cap == 0.f) return launch<T, D, kNoCap>(a, bias, qparts, kparts, st);
  if constexpr (sizeof(T) == 2)
    if (shifted_cap<T>(a.cap)) return launch<T, D, kShiftedCap>(a, bias, qparts, kparts, st);
  return launch<T, D, kExactCap>(a, bias, qparts, kparts, st);
}

template <typename T, int NE>
int run_columns(const Args& a, const Bias& bias, int qparts, int kparts, hipStream_t st) {
  switch (padded(a.d)) {
    case 32: return run_width<T, 32>(a, BiasOf<NE>{bias}, qparts, kparts, st);
    case 64: return run_width<T, 64>(a, BiasOf<NE>{bias}, qparts, kparts, st);
    default: return run_width<T, 128>(a, BiasOf<NE>{bias}, qparts, kparts, st);
  }
}

}  // namespace
}  // namespace attn
}  // namespace ctmr

#define CTMR_BIASED_GRADIENTS(T)                                                                                     \
  template <>                                                                                                        \
  int ctmr::attn::run_biased_gradients<T>(const Args& a, const Bias& bias, bool narrow, int qparts, int kparts,      \
                                          hipStream_t st) {                                                          \
    return narrow ? run_columns<T, 2>(a, bias, qparts, kparts, st) : run_columns<T, 4>(a, bias, qparts, kparts, st); \
  }
