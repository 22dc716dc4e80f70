// V neighbouring elements from float registers to global memory, in one access where V elements are 8 or 16 bytes (the address then has that
// alignment).
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace kfb {

template <int V>
__device__ __forceinline__ void store_vec(float* p, const float* v) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    static_assert(V == 1, "pieces of 1 or a multiple of 4");
    *p = v[0];
  }
}
__device__ __forceinline__ uint32_t bf16_pair_of(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
template <int V>
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float* v) {
  if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair_of(v[0], v[1]), bf16_pair_of(v[2], v[3]), bf16_pair_of(v[4], v[5]), bf16_pair_of(v[6], v[7]));
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pair_of(v[0], v[1]), bf16_pair_of(v[2], v[3]));
  } else {
    static_assert(V == 1, "pieces of 1, 4 or 8");
    *p = __float2bfloat16_rn(v[0]);
  }
}

}  // namespace kfb
