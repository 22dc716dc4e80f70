// Rows of up to 1024 channels, eight a lane: what the kernels of the residual stream share (residual_norm.cu, residual_norm_grad.cu, compress.cu).
//
// A row is held by a team of 8 ... 128 lanes, each with eight neighbouring channels; teams of up to 32 lanes share a warp, larger ones are whole
// warps that meet at a barrier of their own.  A lane's piece is 16 or 32 bytes of bf16 or float32, or 8 bytes of a row kept in 8 bits.
//
// Rows in 8 bits: 32 neighbouring channels share a power of two.  A value is q 2^(e - 133), q a whole number of -127 ... 127, e a byte:
// the exponent field of the group's largest magnitude as a float32, one more where that magnitude would round to 128.  So a value is off by at
// most half a step, 2^-7 of the group's largest, and what comes back is exact in bf16.  e = 255: a value of the group was not finite, and all of them
// come back as NaN.  Groups whose largest magnitude is below 2^-119 (e < 8) come back as zeros with e = 0; e stops at 254, whose values end at 127 2^121.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "vec_io.cuh"

namespace kfb {

constexpr int kPiece = 8;         // channels of a lane
constexpr int kGroup8 = 32;       // channels that share an exponent

__host__ __device__ inline int groups8(int c) { return (c + kGroup8 - 1) / kGroup8; }

// The exponent byte of a group whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t exponent8(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const uint32_t e = (top + 0x10000u) >> 23;
  return e < 8u ? 0u : e > 254u ? 254u : e;
}
__device__ __forceinline__ float step8(uint32_t e) { return e == 255u ? __uint_as_float(0x7fc00000u) : e == 0u ? 0.f : __uint_as_float((e - 6u) << 23); }
// What values are multiplied by before they are rounded.
__device__ __forceinline__ float inverse_step8(uint32_t e) { return e == 255u || e == 0u ? 0.f : __uint_as_float((260u - e) << 23); }

// Four whole numbers as bytes: adding 1.5 2^23 rounds to the nearest (ties to even) and leaves the number in the low byte.
__device__ __forceinline__ uint32_t bytes8(const float* v, float inverse) {
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = fminf(fmaxf(v[i] * inverse, -127.f), 127.f);
    q[i] = __float_as_uint(t + 12582912.f);
  }
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}
// ... and back: a byte with its sign turned round in the low byte of 2^23 is 2^23 + 128 + q.
__device__ __forceinline__ void values8(uint32_t bytes, float step, float* v) {
  const uint32_t t = bytes ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (__uint_as_float(__byte_perm(t, 0x4b000000u, 0x7650 | i)) - 8388736.f) * step;
}

// A lane's eight channels as they lie in memory, of which `n` are there.  VEC: n is 0 or 8 and the address on a 16-byte boundary (8 for bytes).
template <typename T, bool VEC>
struct Piece {
  static constexpr int kWords = kPiece * static_cast<int>(sizeof(T)) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p, int n) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 t = n > 0 ? reinterpret_cast<const uint4*>(p)[i / 4] : make_uint4(0, 0, 0, 0);
        w[i] = t.x;
        w[i + 1] = t.y;
        w[i + 2] = t.z;
        w[i + 3] = t.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) w[i] = i < n ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
    } else {
      const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < kPiece; i += 2) {
        const uint32_t lo = i < n ? s[i] : 0u, hi = i + 1 < n ? s[i + 1] : 0u;
        w[i / 2] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void values(float* v) const {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
      else v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
  }
  // A piece on its way through shared memory (see Ring), and bytes with the word of exponents that theirs lies in.
  __device__ __forceinline__ void take(const uint4* slot, int stride) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 t = slot[i / 4 * stride];
      w[i] = t.x;
      w[i + 1] = t.y;
      w[i + 2] = t.z;
      w[i + 3] = t.w;
    }
  }
  __device__ __forceinline__ void take8(const uint4* slot, int shift) {
    const uint4 t = *slot;
    w[0] = t.x;
    w[1] = t.y;
    w[2] = t.z >> shift & 255u;
  }
  // Bytes and their exponent in the same registers.
  __device__ __forceinline__ void load8(const uint8_t* p, const uint8_t* e, int n) {
    if constexpr (VEC) {
      const uint2 t = n > 0 ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
      w[0] = t.x;
      w[1] = t.y;
    } else {
      w[0] = w[1] = 0u;
#pragma unroll
      for (int i = 0; i < kPiece; ++i)
        if (i < n) w[i / 4] |= static_cast<uint32_t>(p[i]) << 8 * (i & 3);
    }
    w[2] = n > 0 ? *e : 0u;
  }
  __device__ __forceinline__ void values_of_8(float* v) const {
    const float step = step8(w[2]);
    values8(w[0], step, v);
    values8(w[1], step, v + 4);
  }
};

// The first n of eight values to memory.
template <bool VEC, typename T>
__device__ __forceinline__ void store_piece(T* p, const float* v, int n) {
  if constexpr (VEC) {
    if (n > 0) store_vec<kPiece>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < n) store_vec<1>(p + i, v + i);
  }
}

// A lane's eight values (zeros where the row has ended) into bytes and, by the first lane of a group, its exponent.  Four neighbouring lanes hold a group.
template <bool VEC>
__device__ __forceinline__ void store_piece8(uint8_t* p, uint8_t* e, const float* v, int n, bool first) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < kPiece; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t ex = exponent8(top);
  const float inverse = inverse_step8(ex);
  uint32_t q[2] = {bytes8(v, inverse), bytes8(v + 4, inverse)};
  if (ex == 255u) q[0] = q[1] = 0u;      // (what is not finite times zero is no number)
  if constexpr (VEC) {
    if (n > 0) *reinterpret_cast<uint2*>(p) = make_uint2(q[0], q[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
      if (i < n) p[i] = static_cast<uint8_t>(q[i / 4] >> 8 * (i & 3));
  }
  if (first && n > 0) *e = static_cast<uint8_t>(ex);
}

// Copies of 16, 8 or 4 bytes into shared memory that arrive while the thread goes on; zeros where `there` is false.
__device__ __forceinline__ void copy_async16(void* to, const void* from, bool there) {
  const int n = there ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "r"(n) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool there) {
  const int n = there ? BYTES : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_async_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

// Threads of a block and teams in it.
template <int LANES>
struct Teams {
  static constexpr int kGroupLanes = LANES < 32 ? 32 : LANES;        // a warp of small teams, or a large team: what moves from row to row together
  static constexpr int kThreads = LANES == 96 ? 288 : 256;
  static constexpr int kGroups = kThreads / kGroupLanes, kTeams = kGroupLanes / LANES;
  static constexpr int kWarps = LANES < 32 ? 1 : LANES / 32;
};

// Sums of K values over a team's lanes, the same in all of them and in the same order each time.  `turn` alternates from call to call: a buffer is
// written again only behind the barrier of the call between, which every reader of it has passed.
template <int LANES, int K>
__device__ __forceinline__ void team_sum(float (&v)[K], float (*room)[Teams<LANES>::kGroups][Teams<LANES>::kWarps][K], int group, int turn) {
#pragma unroll
  for (int m = (LANES < 32 ? LANES : 32) / 2; m > 0; m >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
  if constexpr (LANES > 32) {
    const int in_team = static_cast<int>(threadIdx.x) % LANES, warp = in_team / 32;
    if (in_team % 32 == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) room[turn][group][warp][k] = v[k];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(LANES) : "memory");
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = room[turn][group][0][k];
#pragma unroll
      for (int w = 1; w < LANES / 32; ++w) t += room[turn][group][w][k];
      v[k] = t;
    }
  }
}

// sigmoid(a) to float32's own rounding, for sums that are stored and then put away in 8 bits: where the sum lies near a border between two stored values, an
// error of the fast exponential (some 2^-21) decides ten times as often as rounding does.  exp(y) by its Taylor series to y^7 / 7! for |y| <= ln 2 / 2
// (the rest is below 2^-27), the powers of two apart.
__device__ __forceinline__ float open_exact(float a) {
  const float x = -fabsf(a), k = rintf(x * 1.44269504f);
  const float y = fmaf(k, -3.19461849e-5f, fmaf(k, -0.693115234375f, x));      // x - k ln 2, ln 2 in two parts, the first of 12 bits
  float t = 1.f / 5040.f;
  t = fmaf(t, y, 1.f / 720.f);
  t = fmaf(t, y, 1.f / 120.f);
  t = fmaf(t, y, 1.f / 24.f);
  t = fmaf(t, y, 1.f / 6.f);
  t = fmaf(t, y, 0.5f);
  t = fmaf(t, y, 1.f);
  t = fmaf(t, y, 1.f);
  const float e = x < -87.f ? 0.f : t * __uint_as_float(static_cast<uint32_t>(static_cast<int>(k) + 127) << 23);
  const float d = __frcp_rn(1.f + e);
  return a < 0.f ? e * d : d;
}

// sigmoid(a) and its slope, from exp(-|a|): 1 - sigmoid(a) by subtraction would lose the slope of an open gate.
struct Gate {
  float open, slope;
};
__device__ __forceinline__ Gate gate_at(float a) {
  const float e = __expf(-fabsf(a)), d = __fdividef(1.f, 1.f + e);
  return {a < 0.f ? e * d : d, e * d * d};
}

}  // namespace kfb
