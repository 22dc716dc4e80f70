// What follows (or goes before) the products of a linear layer, element by element: bias, activation, residual, and their gradient.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#ifdef __CUDACC__
#include "ptx.cuh"
#endif

namespace kfb {

enum Activation : int { kIdentity = 0, kSigmoid = 1, kSilu = 2, kGelu = 3, kRelu = 4 };

#ifdef __CUDACC__
// The activations work on pairs of float32, which the two-wide instructions take at one issue slot a pair: an element's tail, not its products, is what a tile's time
// would be otherwise.  Exponentials and reciprocals are the fast ones and gelu's tail a fit, in float32 compute too: with |z| below 1, sigmoid and silu are within 4 units of
// 2^-24 (elementary float32 operations 3), their slopes 5 (5), gelu 16 (3); z itself is off by more.  Results of float32 layers, gelu, in the root mean square, and those of
// elementary float32 operations: 3 001 rows of 32 -> 384, y 1.0e-7 (1.1e-7), dx 2.5e-7 (3.6e-7), db 2.4e-7 (1.3e-7); 384 -> 384, y 1.6e-7 (3.5e-7), dx 2.6e-7 (4.0e-7), db 2.3e-7 (2.2e-7).
__device__ __forceinline__ uint64_t pair_of(float a) { return ptx::pack2(a, a); }
template <typename F>
__device__ __forceinline__ uint64_t each_of(uint64_t v, F f) {
  const float2 t = ptx::unpack2(v);
  return ptx::pack2(f(t.x), f(t.y));
}
__device__ __forceinline__ uint64_t magnitude(uint64_t v) { return v & 0x7fffffff7fffffffull; }
__device__ __forceinline__ uint64_t reciprocal(uint64_t v) {
  return each_of(v, [](float a) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
  });
}
// 2^v
__device__ __forceinline__ uint64_t power(uint64_t v) {
  return each_of(v, [](float a) { return exp2f(a); });
}
// low where z is negative, high elsewhere
__device__ __forceinline__ uint64_t by_sign(uint64_t z, uint64_t low, uint64_t high) {
  const float2 a = ptx::unpack2(z), l = ptx::unpack2(low), h = ptx::unpack2(high);
  return ptx::pack2(a.x < 0.f ? l.x : h.x, a.y < 0.f ? l.y : h.y);
}

// Phi(-|z|) and exp(-z^2 / 2) for gelu = z Phi(z):  Phi(-|z|) = exp(-z^2 / 2) t P(t), t = 1 / (1 + 0.26517 |z|), P of degree 6 fitted to erfcx by least squares with weights
// that level the relative error, 7e-7 at most for |z| < 13.4, where exp(-z^2 / 2) ends: it keeps its digits where it is small.  size: |z|, finite, so that nothing
// times it is nothing.
__device__ __forceinline__ uint64_t finite_size(uint64_t z) {
  return each_of(magnitude(z), [](float a) { return a > 1e30f ? 1e30f : a; });      // (what is no number stays none)
}
__device__ __forceinline__ uint64_t normal_tail(uint64_t z, uint64_t size, uint64_t& density) {
  density = power(ptx::mul2(ptx::mul2(z, z), pair_of(-0.72134752f)));
  const uint64_t t = reciprocal(ptx::fma2(size, pair_of(0.26516503f), pair_of(1.f)));
  uint64_t p = pair_of(-0.067547895f);
  p = ptx::fma2(p, t, pair_of(0.19396849f));
  p = ptx::fma2(p, t, pair_of(-0.064797565f));
  p = ptx::fma2(p, t, pair_of(0.14152952f));
  p = ptx::fma2(p, t, pair_of(0.08333303f));
  p = ptx::fma2(p, t, pair_of(0.107844375f));
  p = ptx::fma2(p, t, pair_of(0.10566975f));
  return ptx::mul2(ptx::mul2(p, t), density);
}
// sigmoid(z), and its slope from exp(-|z|), so that this stays exact where the gate is open.
__device__ __forceinline__ uint64_t sigmoid_of(uint64_t z, uint64_t& slope) {
  const uint64_t e = power(ptx::mul2(magnitude(z), pair_of(-1.44269504f))), d = reciprocal(ptx::add2(e, pair_of(1.f))), low = ptx::mul2(e, d);
  slope = ptx::mul2(low, d);
  return by_sign(z, low, d);
}

// f(z) and f'(z); gelu is z Phi(z).
template <int ACT>
__device__ __forceinline__ uint64_t activation(uint64_t z) {
  uint64_t other;
  if constexpr (ACT == kRelu) return each_of(z, [](float a) { return a > 0.f || a != a ? a : 0.f; });
  if constexpr (ACT == kGelu) {                      // max(z, 0) - |z| Phi(-|z|)
    const uint64_t size = finite_size(z), low = normal_tail(z, size, other);
    return ptx::fma2(size | 0x8000000080000000ull, low, each_of(z, [](float a) { return fmaxf(a, 0.f); }));
  }
  if constexpr (ACT == kSigmoid) return sigmoid_of(z, other);
  if constexpr (ACT == kSilu) return ptx::mul2(z, sigmoid_of(z, other));
  return z;
}
template <int ACT>
__device__ __forceinline__ uint64_t slope(uint64_t z) {
  uint64_t other;
  if constexpr (ACT == kRelu) return each_of(z, [](float a) { return a > 0.f ? 1.f : 0.f; });
  if constexpr (ACT == kGelu) {
    const uint64_t size = finite_size(z), low = normal_tail(z, size, other);
    const uint64_t v = ptx::fma2(ptx::mul2(size, pair_of(-0.39894228f)), other, low);      // at -|z|: Phi - |z| phi; the slope at |z| is one less that
    return by_sign(z, v, ptx::fma2(v, pair_of(-1.f), pair_of(1.f)));
  }
  if constexpr (ACT == kSigmoid) {
    sigmoid_of(z, other);
    return other;
  }
  if constexpr (ACT == kSilu) {
    const uint64_t s = sigmoid_of(z, other);
    return ptx::fma2(z, other, s);
  }
  return pair_of(1.f);
}

// Sums over a warp's rows (lanes) of eight columns: lane l has column 4 (l >> 4 & 1) + 2 (l >> 3 & 1) + (l >> 2 & 1) at the end.  (Half of the columns change hands
// at each of the first three steps.)
__device__ __forceinline__ float sum_rows8(const uint64_t (&pairs)[4], int lane) {
  float v[8], a[4], b[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = ptx::unpack2(pairs[i]);
    v[2 * i] = t.x;
    v[2 * i + 1] = t.y;
  }
  const bool h4 = lane & 16, h3 = lane & 8, h2 = lane & 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = (h4 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, h4 ? v[i] : v[4 + i], 16);
#pragma unroll
  for (int i = 0; i < 2; ++i) b[i] = (h3 ? a[2 + i] : a[i]) + __shfl_xor_sync(0xffffffffu, h3 ? a[i] : a[2 + i], 8);
  float c = (h2 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, h2 ? b[0] : b[1], 4);
  c += __shfl_xor_sync(0xffffffffu, c, 2);
  return c + __shfl_xor_sync(0xffffffffu, c, 1);
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
int linear_pair_partials(long long rows, int n);       // rows of partial sums
int launch_linear_pair(cudaStream_t stream, const LinearPair& p, const char* tag);

// dW planes: plane[s][n][k] = sum over a piece of the rows of dz^T x (linear_weights.cu).
// add: to what the planes hold.  bias_planes: null, or [linear_weights_bias_planes][n] sums of dz, over rows that are divided between them (not with add).
bool linear_weights_ok(long long rows, int n, int k, bool with_bias);
int linear_weights_splits(long long rows, int n, int k);
int linear_weights_bias_planes(int splits, int k);
int launch_linear_weights(cudaStream_t stream, const void* dz, const void* x, float* planes, float* bias_planes, int splits, int add, long long rows, int n,
                          int k);

}  // namespace kfb
