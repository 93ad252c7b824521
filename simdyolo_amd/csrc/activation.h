// Activations of the normalisation and the gated projections (SY_ACT_*), in
// float32.
#pragma once

#include "parts.h"

namespace sy {

// v / (1 + e^-u), by e^-|u|: nothing overflows, and what is divided by lies
// between 1 and 2, where the hardware's reciprocal is within 1 ulp.
__device__ __forceinline__ float logistic_times(float v, float u) {
  const float e = exp_neg(-__builtin_fabsf(u));
  return v * (u < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e);
}

// `act` is the same in every lane.
__device__ __forceinline__ float activate(int act, float v) {
  switch (act) {
    case SY_ACT_SILU:
      return logistic_times(v, v);
    case SY_ACT_GELU:  // the complement keeps its precision where 1 + erf would lose it
      return 0.5f * v * erfcf(v * -0.70710678f);
    case SY_ACT_GELU_TANH:  // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
      return logistic_times(v, 1.5957691216f * __builtin_fmaf(0.044715f * v * v, v, v));
    case SY_ACT_RELU:
      return v < 0.f ? 0.f : v;  // NaN stays
    case SY_ACT_SIGMOID:
      return logistic_times(1.f, v);
    default:
      return v;
  }
}

}  // namespace sy
