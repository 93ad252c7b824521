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

// N values in registers.  `act` is the same in every lane, and asked for once: a switch at every value costs
// more than most activations.
template <int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
  switch (act) {
    case SY_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = logistic_times(v[i], v[i]);
      return;
    case SY_ACT_GELU:  // the complement keeps its precision where 1 + erf would lose it
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * erfcf(v[i] * -0.70710678f);
      return;
    case SY_ACT_GELU_TANH:  // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
#pragma unroll
      for (int i = 0; i < N; ++i)
        v[i] = logistic_times(v[i], 1.5957691216f * __builtin_fmaf(0.044715f * v[i] * v[i], v[i], v[i]));
      return;
    case SY_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // NaN stays
      return;
    case SY_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = logistic_times(1.f, v[i]);
      return;
  }
}

}  // namespace sy
