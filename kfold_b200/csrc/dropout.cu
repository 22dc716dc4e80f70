// Dropout whose mask is computed from a counter and never stored:  out = (residual +) (kept ? scale x : 0), scale = 1 / (1 - p).  The backward pass is the same
// call on the gradient.
//
// Random words: Philox-4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011),
// key = seed, counter = (e / 4, offset), element e of the mask takes word e % 4 and is dropped when the word is below p 2^32.  So the mask hangs
// on (seed, offset, element) alone: not on the launch shape, the type, or where the tensor lies.
//
// What bounds it: the generator, where every element draws.  Ten rounds are 20 wide multiplications and 20 three-way xors for four words; with the
// comparisons, loads and conversions 24 instructions an element, and the integer pipe, which has the xors and comparisons, is the busiest (63 %; the issue
// slots 65).  384 x 384 x 256 bf16 elements: 44 us with residual, where its 226 MB take 35, and 42 without, where they take 23.  (The comparison as a
// multiply-add, to relieve that pipe: 90 us the two where they are 84; wide multiply-adds run at half the rate.)
// A mask shared along one axis (rows or columns of the pair tensor) is computed once for the positions a thread walks along that axis, and HBM bounds it:
// 768 x 768 x 128, columns, 130 us with residual and its gradient, 755 MB at 5.8 TB/s (a copy has 6.5).
#include <cuda_bf16.h>

#include <type_traits>

#include "ops_common.cuh"
#include "vec_io.cuh"

namespace kfb {
namespace {

constexpr int kThreads = 256;

struct Words {
  uint32_t w[4];
};

// What a launch's words have in common: the seed as the ten rounds' keys, and the products of the first two rounds that hang on the offset alone (the
// second one's on the block's upper half too, which is zero up to 2^34 elements).  STATE: read from device memory when the kernel runs; otherwise
// launch parameters, operands that cost no instruction.
constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u;
struct Stream {
  uint32_t key[20];
  uint32_t offset_hi, b1_hi, b1_lo;      // 64-bit product of the first round with the offset's lower half
  uint32_t a2_hi, a2_lo;                 // of the second round, for an upper half of zero
};
__host__ __device__ __forceinline__ void make_stream(unsigned long long seed, unsigned long long offset, Stream& d) {
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    d.key[2 * i] = k0;
    d.key[2 * i + 1] = k1;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const unsigned long long b1 = static_cast<unsigned long long>(kM1) * static_cast<uint32_t>(offset);
  d.offset_hi = static_cast<uint32_t>(offset >> 32);
  d.b1_hi = static_cast<uint32_t>(b1 >> 32);
  d.b1_lo = static_cast<uint32_t>(b1);
  const unsigned long long a2 = static_cast<unsigned long long>(kM0) * (d.b1_hi ^ d.key[0]);
  d.a2_hi = static_cast<uint32_t>(a2 >> 32);
  d.a2_lo = static_cast<uint32_t>(a2);
}

__device__ __forceinline__ Words philox(unsigned long long block, const Stream& s) {
  const uint32_t upper = static_cast<uint32_t>(block >> 32);
  // the first two rounds
  const unsigned long long a1 = static_cast<unsigned long long>(kM0) * static_cast<uint32_t>(block);
  const uint32_t d2 = static_cast<uint32_t>(a1 >> 32) ^ s.offset_hi ^ s.key[1], d3 = static_cast<uint32_t>(a1);
  uint32_t a2_hi = s.a2_hi, a2_lo = s.a2_lo;
  if (upper != 0) {
    const unsigned long long a2 = static_cast<unsigned long long>(kM0) * (s.b1_hi ^ upper ^ s.key[0]);
    a2_hi = static_cast<uint32_t>(a2 >> 32);
    a2_lo = static_cast<uint32_t>(a2);
  }
  const unsigned long long b2 = static_cast<unsigned long long>(kM1) * d2;
  uint32_t c0 = static_cast<uint32_t>(b2 >> 32) ^ s.b1_lo ^ s.key[2], c1 = static_cast<uint32_t>(b2);
  uint32_t c2 = a2_hi ^ d3 ^ s.key[3], c3 = a2_lo;
#pragma unroll
  for (int i = 2; i < 10; ++i) {
    const unsigned long long a = static_cast<unsigned long long>(kM0) * c0, b = static_cast<unsigned long long>(kM1) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ s.key[2 * i];
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ s.key[2 * i + 1];
    c3 = static_cast<uint32_t>(a);
  }
  return {{c0, c1, c2, c3}};
}

struct DropParams {
  const long long* rng;             // (seed, offset) in device memory, or null: `stream` is made of them
  Stream stream;
  uint32_t cut;                     // kept: word > cut
  int keep_all;                     // nothing is dropped
  float scale;
  long long outer, shared, inner;   // x is [outer][shared][inner], the mask [outer][inner]
  long long chunks, chunk;          // `shared` positions in `chunks` pieces of `chunk`
};

// V elements of x as they lie in memory, and the mask as words to and them with: an element that is dropped becomes a zero whatever it was, an
// infinity or NaN too, at one instruction for two bf16 elements.
template <typename TX, int V>
struct Piece {
  static constexpr int kWords = V * sizeof(TX) < 4 ? 1 : V * static_cast<int>(sizeof(TX)) / 4;
  uint32_t w[kWords];
};
template <typename TX, int V>
__device__ __forceinline__ void load_piece(const TX* p, Piece<TX, V>& d) {
  constexpr int kBytes = V * static_cast<int>(sizeof(TX));
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) {
      const uint4 t = reinterpret_cast<const uint4*>(p)[i];
      d.w[4 * i] = t.x;
      d.w[4 * i + 1] = t.y;
      d.w[4 * i + 2] = t.z;
      d.w[4 * i + 3] = t.w;
    }
  } else if constexpr (kBytes == 8) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    d.w[0] = t.x;
    d.w[1] = t.y;
  } else if constexpr (kBytes == 4) {
    d.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    d.w[0] = *reinterpret_cast<const unsigned short*>(p);
  }
}
template <typename TX, int V>
__device__ __forceinline__ void values(const Piece<TX, V>& d, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (sizeof(TX) == 4) v[i] = __uint_as_float(d.w[i]);
    else v[i] = __uint_as_float(i & 1 ? d.w[i / 2] & 0xffff0000u : d.w[i / 2] << 16);
  }
}

// The mask of elements e ... e + V - 1 (e a multiple of 4 unless V is 1).
template <typename TX, int V>
__device__ __forceinline__ void kept(const DropParams& p, const Stream& stream, long long e, Piece<TX, V>& m) {
#pragma unroll
  for (int i = 0; i < Piece<TX, V>::kWords; ++i) m.w[i] = 0;
  if constexpr (V == 1) {
    const Words r = philox(static_cast<unsigned long long>(e) >> 2, stream);
    const int at = static_cast<int>(e & 3);
    const uint32_t w = at == 0 ? r.w[0] : at == 1 ? r.w[1] : at == 2 ? r.w[2] : r.w[3];
    m.w[0] = (w > p.cut) | p.keep_all ? 0xffffffffu : 0u;
  } else {
#pragma unroll
    for (int b = 0; b < V / 4; ++b) {
      const Words r = philox((static_cast<unsigned long long>(e) >> 2) + b, stream);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 4 * b + i;
        if constexpr (sizeof(TX) == 4) m.w[k] = r.w[i] > p.cut ? 0xffffffffu : 0u;
        else m.w[k / 2] |= r.w[i] > p.cut ? (k & 1 ? 0xffff0000u : 0xffffu) : 0u;
      }
    }
    if (p.keep_all) {
#pragma unroll
      for (int i = 0; i < Piece<TX, V>::kWords; ++i) m.w[i] = 0xffffffffu;
    }
  }
}

// U pieces, their loads before the first store: out may be x or resid, so the compiler keeps the order it is given.  mask(u): the piece's.
template <int V, int U, bool RESID, typename TX, typename TR, typename Mask>
__device__ __forceinline__ void apply(const TX* x, const TR* resid, TR* out, const long long (&at)[U], const bool (&live)[U], float scale, Mask mask) {
  Piece<TX, V> v[U];
  Piece<TR, V> r[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (live[u]) {
      load_piece<TX, V>(x + at[u], v[u]);
      if (RESID) load_piece<TR, V>(resid + at[u], r[u]);
    }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (live[u]) {
      const Piece<TX, V> m = mask(u);
#pragma unroll
      for (int i = 0; i < Piece<TX, V>::kWords; ++i) v[u].w[i] &= m.w[i];
      float f[V], add[V];
      values<TX, V>(v[u], f);
      if (RESID) values<TR, V>(r[u], add);
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = RESID ? fmaf(f[i], scale, add[i]) : f[i] * scale;
      store_vec<V>(out + at[u], f);
    }
}

constexpr int kBlocksPerSm = 4;

// Every element by itself: `inner` of them, a multiple of V.
template <typename TX, typename TR, int V, bool RESID, bool STATE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) dropout_kernel(const TX* x, const TR* resid, TR* out, const DropParams p) {
  constexpr int U = 2;
  grid_dependency_enter();
  Stream own;
  if (STATE) make_stream(static_cast<unsigned long long>(p.rng[0]), static_cast<unsigned long long>(p.rng[1]), own);
  const Stream& stream = STATE ? own : p.stream;
  constexpr long long kBlock = static_cast<long long>(kThreads) * U * V;
  for (long long base = blockIdx.x * kBlock; base < p.inner; base += gridDim.x * kBlock) {
    long long at[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = base + (u * kThreads + static_cast<int>(threadIdx.x)) * V;
      live[u] = at[u] < p.inner;
    }
    apply<V, U, RESID>(x, resid, out, at, live, p.scale, [&](int u) {
      Piece<TX, V> m;
      kept<TX, V>(p, stream, at[u], m);
      return m;
    });
  }
}

// A shared mask: a thread has V elements of it and the positions of its piece of the shared axis.
template <typename TX, typename TR, int V, bool RESID, bool STATE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) dropout_shared_kernel(const TX* x, const TR* resid, TR* out, const DropParams p) {
  constexpr int U = RESID ? 3 : 4;
  grid_dependency_enter();
  Stream own;
  if (STATE) make_stream(static_cast<unsigned long long>(p.rng[0]), static_cast<unsigned long long>(p.rng[1]), own);
  const Stream& stream = STATE ? own : p.stream;
  const long long pieces = p.inner / V, total = p.outer * p.chunks * pieces;
  for (long long t = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; t < total; t += static_cast<long long>(gridDim.x) * kThreads) {
    const long long i = t % pieces * V, rest = t / pieces, o = rest / p.chunks, s0 = rest % p.chunks * p.chunk;
    // (a piece of the shared axis is short, or the threads are many: either way below 2^31 for what a GPU can hold)
    int left = static_cast<int>(s0 + p.chunk < p.shared ? p.chunk : p.shared - s0);
    Piece<TX, V> m;
    kept<TX, V>(p, stream, o * p.inner + i, m);
    const long long first = (o * p.shared + s0) * p.inner + i;
    const TX* xs = x + first;
    const TR* rs = RESID ? resid + first : nullptr;
    TR* os = out + first;
    for (; left > 0; left -= U) {
      long long at[U];
      bool live[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        at[u] = u * p.inner;
        live[u] = u < left;
      }
      apply<V, U, RESID>(xs, rs, os, at, live, p.scale, [&](int) { return m; });
      xs += U * p.inner;
      if (RESID) rs += U * p.inner;
      os += U * p.inner;
    }
  }
}

template <typename TX, typename TR, int V, bool RESID, bool STATE>
int launch_state(cudaStream_t stream, const void* x, const void* resid, void* out, DropParams p) {
  const long long sms = sm_count();
  LaunchScope scope(stream, "dropout");
  if (p.shared == 1) {
    p.inner *= p.outer;
    const long long blocks = (p.inner + 2ll * V * kThreads - 1) / (2ll * V * kThreads);
    return launch_kernel(stream, dropout_kernel<TX, TR, V, RESID, STATE>, static_cast<unsigned>(blocks < sms * 64 ? blocks : sms * 64), kThreads, 0,
                         static_cast<const TX*>(x), static_cast<const TR*>(resid), static_cast<TR*>(out), p);
  }
  // pieces of the shared axis: as many as fill the device once
  const long long items = p.outer * (p.inner / V), full = sms * kBlocksPerSm * kThreads;
  long long chunks = items >= full ? 1 : full / items;
  if (chunks > p.shared) chunks = p.shared;
  p.chunk = (p.shared + chunks - 1) / chunks;
  p.chunks = (p.shared + p.chunk - 1) / p.chunk;
  const long long blocks = (items * p.chunks + kThreads - 1) / kThreads;
  return launch_kernel(stream, dropout_shared_kernel<TX, TR, V, RESID, STATE>, static_cast<unsigned>(blocks < sms * 64 ? blocks : sms * 64), kThreads, 0,
                       static_cast<const TX*>(x), static_cast<const TR*>(resid), static_cast<TR*>(out), p);
}
template <typename TX, typename TR, int V, bool RESID>
int launch_resid(cudaStream_t stream, const void* x, const void* resid, void* out, const DropParams& p) {
  return p.rng != nullptr ? launch_state<TX, TR, V, RESID, true>(stream, x, resid, out, p) : launch_state<TX, TR, V, RESID, false>(stream, x, resid, out, p);
}
template <typename TX, typename TR, int V>
int launch(cudaStream_t stream, const void* x, const void* resid, void* out, const DropParams& p) {
  return resid != nullptr ? launch_resid<TX, TR, V, true>(stream, x, resid, out, p) : launch_resid<TX, TR, V, false>(stream, x, resid, out, p);
}

template <typename TX, typename TR>
int dispatch(cudaStream_t stream, const void* x, const void* resid, void* out, const DropParams& p) {
  constexpr int V = std::is_same<TX, __nv_bfloat16>::value && std::is_same<TR, __nv_bfloat16>::value ? 8 : 4;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(resid) | reinterpret_cast<uintptr_t>(out);
  const long long run = p.shared == 1 ? p.outer * p.inner : p.inner;      // neighbours in memory whose mask elements are neighbours
  if ((at & 15) == 0 && run % V == 0) return launch<TX, TR, V>(stream, x, resid, out, p);
  if ((at & 15) == 0 && run % 4 == 0) return launch<TX, TR, 4>(stream, x, resid, out, p);
  return launch<TX, TR, 1>(stream, x, resid, out, p);
}

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" KFB_API int kfb_dropout(const void* x, const void* residual, void* out, long long outer, long long shared, long long inner,
                                   long long drop_below, float scale, const long long* rng, long long seed, long long offset, int x_dtype,
                                   int out_dtype, void* stream) {
  KFB_CHECK_ARG(outer >= 0 && shared >= 0 && inner >= 0, "dropout: extents %lld %lld %lld", outer, shared, inner);
  KFB_CHECK_ARG(drop_below >= 0 && drop_below <= (1ll << 32), "dropout: drop_below %lld is not in [0, 2^32]", drop_below);
  KFB_CHECK_ARG((x_dtype == KFB_BF16 || x_dtype == KFB_FP32) && (out_dtype == KFB_FP32 || (out_dtype == KFB_BF16 && x_dtype == KFB_BF16)),
                "dropout: bad dtypes %d -> %d", x_dtype, out_dtype);
  if (outer == 0 || shared == 0 || inner == 0) return KFB_OK;
  KFB_CHECK_ARG(x != nullptr && out != nullptr, "dropout: null tensor");
  DropParams d = {};
  d.rng = rng;
  make_stream(static_cast<unsigned long long>(seed), static_cast<unsigned long long>(offset), d.stream);
  d.keep_all = drop_below == 0;
  d.cut = drop_below == 0 ? 0u : static_cast<uint32_t>(drop_below - 1);
  d.scale = scale;
  d.outer = outer;
  d.shared = shared;
  d.inner = inner;
  cudaStream_t s = as_stream(stream);
  if (x_dtype == KFB_BF16)
    return out_dtype == KFB_BF16 ? dispatch<__nv_bfloat16, __nv_bfloat16>(s, x, residual, out, d) : dispatch<__nv_bfloat16, float>(s, x, residual, out, d);
  return dispatch<float, float>(s, x, residual, out, d);
}
