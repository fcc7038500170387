// Element types of the differentiable operators (fp32, bf16, fp16) and the
// host's checks that they share.
#pragma once

#include "ctmr_common.hpp"

namespace ctmr {

template <typename T, int V>
using Vec = T __attribute__((ext_vector_type(V)));

template <typename T, int V>
__device__ __forceinline__ Vec<float, V> load_as_float(const T* p) {
  return __builtin_convertvector(*reinterpret_cast<const Vec<T, V>*>(p), Vec<float, V>);
}

// Rounds to nearest even where T has 16 bits.
template <typename T, int V>
__device__ __forceinline__ void store_rounded(T* p, const Vec<float, V>& v) {
  *reinterpret_cast<Vec<T, V>*>(p) = __builtin_convertvector(v, Vec<T, V>);
}

// A parameter of any element type (enum ctmr_elem; the type is the same for the
// whole launch), read and written one by one outside the inner loops.
__device__ __forceinline__ float load_param(const void* p, int elem, int64_t i) {
  if (elem == CTMR_ELEM_F32) return static_cast<const float*>(p)[i];
  if (elem == CTMR_ELEM_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_param(void* p, int elem, int64_t i, float v) {
  if (elem == CTMR_ELEM_F32) static_cast<float*>(p)[i] = v;
  else if (elem == CTMR_ELEM_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

inline bool valid_elem(int elem) { return elem >= CTMR_ELEM_F32 && elem <= CTMR_ELEM_F16; }
inline int elem_bytes(int elem) { return elem == CTMR_ELEM_F32 ? 4 : 2; }

}  // namespace ctmr
