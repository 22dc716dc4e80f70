// What follows (or goes before) the products of a linear layer, element by element: bias, activation, residual, and their gradient.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace kfb {

enum Activation : int { kIdentity = 0, kSigmoid = 1, kSilu = 2, kGelu = 3, kRelu = 4 };

#ifdef __CUDACC__
// The complementary error function for x >= 0 by the Chebyshev fit of Press, Teukolsky, Vetterling and Flannery, "Numerical Recipes in C" (1992), 6.2,
// whose relative error is below 1.2e-7 everywhere: Phi(z) keeps its digits where it is small.
__device__ __forceinline__ float erfc_positive(float x) {
  const float t = __fdividef(1.f, fmaf(0.5f, x, 1.f));
  float q = 0.17087277f;
  q = fmaf(q, t, -0.82215223f);
  q = fmaf(q, t, 1.48851587f);
  q = fmaf(q, t, -1.13520398f);
  q = fmaf(q, t, 0.27886807f);
  q = fmaf(q, t, -0.18628806f);
  q = fmaf(q, t, 0.09678418f);
  q = fmaf(q, t, 0.37409196f);
  q = fmaf(q, t, 1.00002368f);
  q = fmaf(q, t, -1.26551223f);
  return t * __expf(fmaf(-x, x, q));
}
__device__ __forceinline__ float normal_cdf(float z) {
  const float t = 0.5f * erfc_positive(0.70710678f * fabsf(z));
  return z < 0.f ? t : 1.f - t;
}

// f(z) and f'(z).  sigmoid's slope comes from exp(-|z|), so that it stays exact where the gate is open; gelu is z Phi(z).
template <int ACT>
__device__ __forceinline__ float activation(float z) {
  if constexpr (ACT == kRelu) return z > 0.f || z != z ? z : 0.f;
  if constexpr (ACT == kGelu) return z * normal_cdf(z);
  if constexpr (ACT == kSigmoid || ACT == kSilu) {
    const float e = __expf(-fabsf(z)), d = __fdividef(1.f, 1.f + e), s = z < 0.f ? e * d : d;
    return ACT == kSigmoid ? s : z * s;
  }
  return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if constexpr (ACT == kRelu) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == kGelu) return fmaf(z * 0.39894228f, __expf(-0.5f * z * z), normal_cdf(z));
  if constexpr (ACT == kSigmoid || ACT == kSilu) {
    const float e = __expf(-fabsf(z)), d = __fdividef(1.f, 1.f + e), s = z < 0.f ? e * d : d, ss = e * d * d;
    return ACT == kSigmoid ? ss : fmaf(z, ss, s);
  }
  return 1.f;
}
// A call with the activation as a constant.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F f) {
  switch (act) {
    case kSigmoid: f(std::integral_constant<int, kSigmoid>()); break;
    case kSilu: f(std::integral_constant<int, kSilu>()); break;
    case kGelu: f(std::integral_constant<int, kGelu>()); break;
    case kRelu: f(std::integral_constant<int, kRelu>()); break;
    default: f(std::integral_constant<int, kIdentity>());
  }
}
#endif

// ---- many rows, bf16 throughout, CTA pairs (linear_pair.cu)
enum Tail : int { kPlainTail = 0, kForwardTail = 1, kBackwardTail = 2 };
struct LinearPair {
  int tail;
  const void* a;             // (rows, k)
  const void* b;             // (n, k), or (k, n) where by_k
  int by_k;
  const float* bias;         // forward and backward: z = a b^T + bias
  int act;
  const void* aux;           // (rows, n): forward the residual or null, backward dy
  void* out;                 // (rows, n): f(z) + aux; aux f'(z); or the products alone
  float* partial;            // backward, or null: [linear_pair_partials][n] sums of out before it is rounded
  long long rows;
  int n, k;
};
bool linear_pair_ok(long long rows, int n, int k);
int linear_pair_partials(long long rows, int n, int k);       // rows of partial sums
int launch_linear_pair(cudaStream_t stream, const LinearPair& p, const char* tag);

// dW planes: plane[s][n][k] = sum over a piece of the rows of dz^T x (linear_weights.cu).
bool linear_weights_ok(int n, int k);
int linear_weights_splits(long long rows, int n, int k);
int launch_linear_weights(cudaStream_t stream, const void* dz, const void* x, float* planes, int splits, int add, long long rows, int n, int k);

}  // namespace kfb
