// Rows of up to 1024 channels in the registers of up to 32 lanes: what the kernels of the residual stream share (residual_norm.cu,
// residual_norm_grad.cu), and rows in 8 bits (compress.cu too).
//
// A team of 8, 16 or 32 lanes holds a row, P pieces of eight neighbouring channels a lane; a piece is 16 or 32 bytes of bf16 or float32, or 8 bytes of a row
// kept in 8 bits, and four pairs of float32 in registers, which the two-wide instructions take at one issue slot a pair.  (One piece a lane, and several warps
// for a wide row, took 375 instructions a warp and row where these rows of 768 channels take a third; issue slots were what bounded them.)
//
// Rows in 8 bits: 32 neighbouring channels share a power of two.  A value is q 2^(e - 133), q a whole number of -127 ... 127, e a byte:
// the exponent field of the group's largest magnitude as a float32, one more where that magnitude would round to 128.  So a value is off by at
// most half a step, 2^-7 of the group's largest, and what comes back is exact in bf16.  e = 255: a value of the group was not finite, and all of them
// come back as NaN.  Groups whose largest magnitude is below 2^-119 (e < 8) come back as zeros with e = 0; e stops at 254, whose values end at 127 2^121.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "ptx.cuh"
#include "vec_io.cuh"

namespace kfb {

constexpr int kPiece = 8;         // channels of a piece
constexpr int kGroup8 = 32;       // channels that share an exponent

__host__ __device__ inline int groups8(int c) { return (c + kGroup8 - 1) / kGroup8; }

struct Pairs {
  uint64_t v[kPiece / 2];
  __device__ __forceinline__ float get(int i) const {
    const float2 f = ptx::unpack2(v[i / 2]);
    return i & 1 ? f.y : f.x;
  }
};
__device__ __forceinline__ Pairs both(float a) {
  const uint64_t t = ptx::pack2(a, a);
  return {{t, t, t, t}};
}
__device__ __forceinline__ Pairs of_floats(const float* f) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < kPiece / 2; ++i) r.v[i] = ptx::pack2(f[2 * i], f[2 * i + 1]);
  return r;
}
__device__ __forceinline__ Pairs of_bf16(const uint4& w) {
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::pack2(q[i] << 16, q[i] & 0xffff0000u);
  return r;
}
__device__ __forceinline__ Pairs of_f32(const uint4& a, const uint4& b) {
  return {{ptx::pack2(a.x, a.y), ptx::pack2(a.z, a.w), ptx::pack2(b.x, b.y), ptx::pack2(b.z, b.w)}};
}
__device__ __forceinline__ uint4 to_bf16(const Pairs& p) {
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = ptx::unpack2(p.v[i]);
    q[i] = bf16_pair_of(f.x, f.y);
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}
__device__ __forceinline__ Pairs add(const Pairs& a, const Pairs& b) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::add2(a.v[i], b.v[i]);
  return r;
}
__device__ __forceinline__ Pairs mul(const Pairs& a, const Pairs& b) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::mul2(a.v[i], b.v[i]);
  return r;
}
__device__ __forceinline__ Pairs fma(const Pairs& a, const Pairs& b, const Pairs& c) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ptx::fma2(a.v[i], b.v[i], c.v[i]);
  return r;
}
// The sum of the elements: of pairs that were added up side by side, so that no addition waits for the one before it.
__device__ __forceinline__ float total(const Pairs& a) {
  const float2 f = ptx::unpack2(ptx::add2(ptx::add2(a.v[0], a.v[1]), ptx::add2(a.v[2], a.v[3])));
  return f.x + f.y;
}
template <typename F>
__device__ __forceinline__ Pairs each(const Pairs& a, F f) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = ptx::unpack2(a.v[i]);
    r.v[i] = ptx::pack2(f(t.x), f(t.y));
  }
  return r;
}

// ---- rows in 8 bits
// The exponent byte of a group whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t exponent8(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const uint32_t e = (top + 0x10000u) >> 23;
  return e < 8u ? 0u : e > 254u ? 254u : e;
}
__device__ __forceinline__ float step8(uint32_t e) { return e == 255u ? __uint_as_float(0x7fc00000u) : e == 0u ? 0.f : __uint_as_float((e - 6u) << 23); }
// What values are multiplied by before they are rounded.
__device__ __forceinline__ float inverse_step8(uint32_t e) { return e == 255u || e == 0u ? 0.f : __uint_as_float((260u - e) << 23); }

// Eight whole numbers as bytes: adding 1.5 2^23 rounds to the nearest (ties to even) and leaves the number in the low byte.
__device__ __forceinline__ uint2 bytes8(const Pairs& p, uint32_t e) {
  const float inverse = inverse_step8(e);
  Pairs t = p;
  if (e == 254u) t = each(p, [](float v) { return fminf(fmaxf(v, __uint_as_float(0xff7e0000u)), __uint_as_float(0x7f7e0000u)); });      // (the one that stops short, at 127 2^121)
  t = fma(t, both(inverse), both(12582912.f));
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = ptx::unpack2(t.v[2 * i]), b = ptx::unpack2(t.v[2 * i + 1]);
    w[i] = __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
  }
  return e == 255u ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);      // (what is not finite times zero is no number)
}
// ... and back: a byte with its sign turned round in the low byte of 2^23 is 2^23 + 128 + q.
__device__ __forceinline__ Pairs values8(const uint2& bytes, uint32_t e) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = (i < 2 ? bytes.x : bytes.y) ^ 0x80808080u, at = 2 * (i & 1);
    r.v[i] = ptx::pack2(__byte_perm(t, 0x4b000000u, 0x7650 | at), __byte_perm(t, 0x4b000000u, 0x7650 | (at + 1)));
  }
  return mul(add(r, both(-8388736.f)), both(step8(e)));
}
// The bits of the largest magnitude of a piece, in float32: of values, or of bf16 words, two at a time.
__device__ __forceinline__ uint32_t top_of(const Pairs& p) {
  uint32_t t = 0u;
#pragma unroll
  for (int i = 0; i < kPiece; ++i) t = max(t, __float_as_uint(p.get(i)) & 0x7fffffffu);
  return t;
}
__device__ __forceinline__ uint32_t top_of(const uint4& w) {
  const uint32_t m = 0x7fff7fffu, t = __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
  return max(t << 16, t & 0xffff0000u);
}
// ... of a group, which four neighbouring lanes hold.
__device__ __forceinline__ uint32_t group_top(uint32_t t) {
  t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
  return max(t, __shfl_xor_sync(0xffffffffu, t, 2));
}

// ---- pieces in memory, of which the first `n` channels are there.  VEC: eight neighbouring channels, n is 0 or 8 and the address on a 16-byte boundary (8 for bytes).
// Otherwise (any width, any address) a lane has every 32nd channel, so that a warp's accesses lie side by side and a group of 32 is the warp's: p, and e of bytes, are
// then those of the lane's first channel; all lanes of a warp come to the bytes together, with one piece of one row.
constexpr int kSpread = 32;
template <bool VEC>
__host__ __device__ constexpr int channel_step() { return VEC ? 1 : kSpread; }
// Channels of a piece that a row of c has, and its first channel.
template <bool VEC>
__device__ __forceinline__ int channels_of(int c, int first) { return min(max(VEC ? c - first : (c - first + kSpread - 1) / kSpread, 0), kPiece); }

template <typename T, bool VEC>
__device__ __forceinline__ Pairs load_piece(const T* p, int n) {
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if constexpr (VEC) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    if constexpr (sizeof(T) == 2) return of_bf16(n > 0 ? q[0] : zero);
    else return of_f32(n > 0 ? q[0] : zero, n > 0 ? q[1] : zero);
  } else {
    float f[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      if constexpr (sizeof(T) == 2) f[i] = i < n ? __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const unsigned short*>(p)[i * kSpread]) << 16) : 0.f;
      else f[i] = i < n ? p[i * kSpread] : 0.f;
    }
    return of_floats(f);
  }
}
template <bool VEC>
__device__ __forceinline__ Pairs load_piece8(const uint8_t* p, const uint8_t* e, int n) {
  if constexpr (VEC) {
    return values8(n > 0 ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0), n > 0 ? *e : 0u);
  } else {
    // (lane i takes the exponent of group i for all)
    uint32_t b[kPiece];
    const int lane = threadIdx.x % 32, most = __shfl_sync(0xffffffffu, n, 0);
    const float step = lane < most && lane < kPiece ? step8(e[lane]) : 0.f;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) b[i] = i < n ? p[i * kSpread] : 0u;
    float f[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) f[i] = static_cast<float>(static_cast<int8_t>(b[i])) * __shfl_sync(0xffffffffu, step, i);
    return of_floats(f);
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_piece(T* p, const Pairs& v, int n) {
  if constexpr (VEC) {
    if (n <= 0) return;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p) = to_bf16(v);
    } else {
      ulonglong2* q = reinterpret_cast<ulonglong2*>(p);
      q[0] = make_ulonglong2(v.v[0], v.v[1]);
      q[1] = make_ulonglong2(v.v[2], v.v[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const float f = v.get(i);
      if (i < n) store_vec<1>(p + i * kSpread, &f);
    }
  }
}
// Values into bytes, and by the first lane of a group its exponent.  `top`: of the piece (VEC).  All lanes of a warp come here together.
template <bool VEC>
__device__ __forceinline__ void store_piece8(uint8_t* p, uint8_t* e, const Pairs& v, uint32_t top, int n, int lane) {
  if constexpr (VEC) {
    const uint32_t ex = exponent8(group_top(top));
    const uint2 q = bytes8(v, ex);
    if (n <= 0) return;
    *reinterpret_cast<uint2*>(p) = q;
    if (lane % (kGroup8 / kPiece) == 0) *e = static_cast<uint8_t>(ex);
  } else {
    // (lane i works out the exponent of group i for all; the first lane has a channel of every group that is there)
    const int lane32 = threadIdx.x % 32, most = __shfl_sync(0xffffffffu, n, 0);
    uint32_t mine = 0u;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const uint32_t t = __reduce_max_sync(0xffffffffu, __float_as_uint(v.get(i)) & 0x7fffffffu);
      if (lane32 == i) mine = t;
    }
    const uint32_t ex = exponent8(mine);
    const float inverse = inverse_step8(ex);
    const uint32_t bad = __ballot_sync(0xffffffffu, ex == 255u);
    if (lane32 < most && lane32 < kPiece) e[lane32] = static_cast<uint8_t>(ex);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const float t = fminf(fmaxf(v.get(i) * __shfl_sync(0xffffffffu, inverse, i), -127.f), 127.f) + 12582912.f;
      if (i < n) p[i * kSpread] = bad >> i & 1u ? 0 : static_cast<uint8_t>(__float_as_uint(t));
    }
  }
}

// ---- copies of 16, 8 or 4 bytes into shared memory that arrive while the thread goes on; zeros where `there` is false
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool there) {
  const int n = there ? BYTES : 0;
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_async_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LATER>
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LATER) : "memory"); }

// ---- gates
// A reciprocal of 1 ... 10^38, rounded correctly by Markstein's step (IBM J. Res. Dev. 34, 1990) from one within a unit.
__device__ __forceinline__ float reciprocal_of(float w) {
  const float d = __fdividef(1.f, w);
  return fmaf(fmaf(-w, d, 1.f), d, d);
}
// A gate with logit a as one number: sigmoid(-|a|), with a's sign.  Both sigmoid(a) and its slope come from it without the subtraction that would
// lose the slope of an open gate.  T: the logits' type.  What bf16 logits open or shut is bf16 too (y and u, or dy, though dx may be
// float32), 2^-9, beside which the fast exponential's 2^-21 is nothing; float32 logits take the exact one, in files that are built with it, and the reciprocal above.
template <typename T>
__device__ __forceinline__ float gate_at(float a) {
  if constexpr (sizeof(T) == 2) {
    const float e = __expf(-fabsf(a));
    return copysignf(__fdividef(e, 1.f + e), a);
  } else {
    const float e = expf(-fabsf(a));
    return copysignf(e * reciprocal_of(1.f + e), a);
  }
}
__device__ __forceinline__ float open_of(float q) { return __float_as_int(q) < 0 ? -q : 1.f - q; }
__device__ __forceinline__ float slope_of(float q) { return fmaf(-q, q, fabsf(q)); }

}  // namespace kfb
