// Device pieces of the attention kernels on the bf16 matrix cores: float32 operands
// as three bf16 parts (attention.hip states the arithmetic), and their exponential.
#pragma once

#include "split.h"

namespace sy {

// e^x for x up to a few units: 2^t of the hardware at t = x log2(e) rounded, times 1 plus the
// first-order term of t's exact rounding error and of log2(e)'s.  Below -150,
// where the result is under every float, 0; NaN stays.
__device__ __forceinline__ float exp_neg(float x) {
  constexpr float kLog2e = 1.4426950408889634f, kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);
  x = x < -150.f ? -150.f : x;
  const float t = x * kLog2e, r = __builtin_fmaf(x, kLog2eLow, __builtin_fmaf(x, kLog2e, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return __builtin_fmaf(p, r * 0.69314718f, p);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight floats as three bf16 parts each, v = p[0] + p[1] + p[2] exactly.
__device__ __forceinline__ void parts8(const f32x4& x, const f32x4& y, bf16x8 (&p)[3]) {
  u32x4 w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x2v v = i < 2 ? f32x2v{x[2 * i], x[2 * i + 1]} : f32x2v{y[2 * i - 4], y[2 * i - 3]};
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      const unsigned b = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
      w[s][i] = b;
      if (s < 2) {
        v[0] -= __builtin_bit_cast(float, b << 16);
        v[1] -= __builtin_bit_cast(float, b & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 3; ++s) p[s] = __builtin_bit_cast(bf16x8, w[s]);
}

// main + rest += a b: the leading parts' product in main, the five next ones in
// rest.
__device__ __forceinline__ void mfma_parts(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x16& main, f32x16& rest) {
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], rest, 0, 0, 0);
  main = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], main, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], rest, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], rest, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], rest, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], rest, 0, 0, 0);
}

}  // namespace sy
