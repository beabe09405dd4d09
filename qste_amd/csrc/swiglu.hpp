// silu(g) * u for one element: as torch's operators round it (the gate's own
// passes), and in one (the products that end in it).
#pragma once

#include "common.hpp"

namespace qste {
namespace swiglu {

__device__ __forceinline__ float silu_value(float x) { return x / (1.0f + expf(-x)); }

template <int DT>
__device__ __forceinline__ float forward_one(float g, float u) {
  using E = Elem<DT>;
  const float a = E::round(silu_value(g));
  return a * u;  // rounded by the caller's store
}

// The same, in bf16 with the hardware's exponential and reciprocal where they leave no
// doubt about the rounding: for |g| < 16 their value is within 30 2^-24 of
// silu_value's (24 from the exponent's rounding), 30 units of its last place, and is
// taken unless it lies within 32 of them of the middle between two bf16 values (one
// in a thousand).  A division and a full exponential less: with the blocks 43 -> 33
// instructions an element; us, 16384 x 14336 391 -> 386, 4096 x 4096 24.1 -> 22.7.
template <int DT>
__device__ __forceinline__ float forward_fast(float g, float u) {
  if constexpr (DT == QSTE_BF16) {
    float a = g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f));
    const uint32_t past = (__float_as_uint(a) - 0x8000u + 32u) & 0xFFFFu;
    if (past < 64u || !(fabsf(g) < 16.0f)) a = silu_value(g);
    return Elem<DT>::round(a) * u;  // rounded by the caller's store
  } else {
    return forward_one<DT>(g, u);
  }
}

// silu(g) u before its only rounding, to the type.  16-bit types leave room for
// the hardware's exponential and reciprocal: within 2^-24 (max(-g, 0) + 11) of the
// value for g > -87, and a third of the instructions (the tiles' 8190 x 14336 over
// 4096: 1373 -> 1261 us).  Below -87, where |silu(g)| < 2^-118, the exponential passes
// fp32's end or its reciprocal the normal numbers, and the value goes to 0 (for
// g < -88.8 silu_value's does too).
template <int DT>
__device__ __forceinline__ float gated_one(float g, float u) {
  if constexpr (DT == QSTE_F32)
    return silu_value(g) * u;
  else
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f)) * u;
}

}  // namespace swiglu
}  // namespace qste
