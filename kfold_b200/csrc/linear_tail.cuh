// What follows (or goes before) the products of a linear layer, element by element: bias, activation, residual, and their gradient.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace kfb {

enum Activation : int { kIdentity = 0, kSigmoid = 1, kSilu = 2, kGelu = 3, kRelu = 4 };

#ifdef __CUDACC__
// f(z) and f'(z).  sigmoid's slope comes from exp(-|z|), so that it stays exact where the gate is open; gelu is z Phi(z) with the error function.
template <int ACT>
__device__ __forceinline__ float activation(float z) {
  if constexpr (ACT == kRelu) return fmaxf(z, 0.f) + (z != z ? z : 0.f);
  if constexpr (ACT == kGelu) return 0.5f * z * erfcf(-0.70710678f * z);
  if constexpr (ACT == kSigmoid || ACT == kSilu) {
    const float e = __expf(-fabsf(z)), d = __fdividef(1.f, 1.f + e), s = z < 0.f ? e * d : d;
    return ACT == kSigmoid ? s : z * s;
  }
  return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if constexpr (ACT == kRelu) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == kGelu) return fmaf(z * 0.39894228f, __expf(-0.5f * z * z), 0.5f * erfcf(-0.70710678f * z));
  if constexpr (ACT == kSigmoid || ACT == kSilu) {
    const float e = __expf(-fabsf(z)), d = __fdividef(1.f, 1.f + e), s = z < 0.f ? e * d : d, ss = e * d * d;
    return ACT == kSigmoid ? ss : fmaf(z, ss, s);
  }
  return 1.f;
}
#endif

}  // namespace kfb
