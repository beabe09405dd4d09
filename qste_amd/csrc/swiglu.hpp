// silu(g) * u for one element, rounded as torch's operators round it: shared by
// the gate's own passes and the products that end in it, so all give the same bits.
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

}  // namespace swiglu
}  // namespace qste
