// The gradients' kernels of the masked attention with a position bias for one type of
// heads, which the including source instantiates.
#pragma once

#include "masked_attention_backward.hpp"

namespace ctmr {
namespace attn {
namespace {

template <typename T, int D, int ST>
int run_width(const Args& a, const BiasOf<ST>& bias, int qparts, int kparts, hipStream_t st) {
  if (a.cap == 0.f) return launch<T, D, kNoCap>(a, bias, qparts, kparts, st);
  if constexpr (sizeof(T) == 2)
    if (shifted_cap<T>(a.cap)) return launch<T, D, kShiftedCap>(a, bias, qparts, kparts, st);
  return launch<T, D, kExactCap>(a, bias, qparts, kparts, st);
}

template <typename T, int ST>
int run_columns(const Args& a, const Bias& bias, int qparts, int kparts, hipStream_t st) {
  switch (padded(a.d)) {
    case 32: return run_width<T, 32>(a, BiasOf<ST>{bias}, qparts, kparts, st);
    case 64: return run_width<T, 64>(a, BiasOf<ST>{bias}, qparts, kparts, st);
    default: return run_width<T, 128>(a, BiasOf<ST>{bias}, qparts, kparts, st);
  }
}

}  // namespace
}  // namespace attn
}  // namespace ctmr

#define CTMR_BIASED_GRADIENTS(T)                                                                                   \
  template <>                                                                                                      \
  int ctmr::attn::run_biased_gradients<T>(const Args& a, const Bias& bias, int steps, int qparts, int kparts,      \
                                          hipStream_t st) {                                                        \
    switch (steps) {                                                                                               \
      case 3: return run_columns<T, 3>(a, bias, qparts, kparts, st);                                               \
      case 4: return run_columns<T, 4>(a, bias, qparts, kparts, st);                                               \
      case 6: return run_columns<T, 6>(a, bias, qparts, kparts, st);                                               \
      default: return run_columns<T, 8>(a, bias, qparts, kparts, st);                                              \
    }                                                                                                              \
  }
