// Dropout whose mask is computed from a counter and never stored:  out = (residual +) (kept ? scale x : 0), scale = 1 / (1 - p).  The backward pass is the same
// call on the gradient.
//
// Random words: Philox-4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011),
// key = seed, counter = (e / 4, offset), element e of the mask takes word e % 4 and is dropped when the word is below p 2^32.  So the mask hangs
// on (seed, offset, element) alone: not on the launch shape, the type, or where the tensor lies.
//
// What bounds it: HBM, as long as the generator stays under it.  Ten rounds are 20 wide multiplications and 20 three-way xors for four words, ten
// instructions an element where the memory's rate leaves 33.  A mask shared along one axis (rows or columns of the pair tensor) is computed
// once for the positions a thread walks along that axis.
#include <cuda_bf16.h>

#include <type_traits>

#include "ops_common.cuh"
#include "vec_io.cuh"

namespace kfb {
namespace {

constexpr int kThreads = 256;

struct DropParams {
  const long long* rng;             // (seed, offset) in device memory, or null: the two below
  unsigned long long seed, offset;
  uint32_t cut;                     // kept: word > cut
  int keep_all;                     // nothing is dropped
  float scale;
  long long outer, shared, inner;   // x is [outer][shared][inner], the mask [outer][inner]
  long long chunks, chunk;          // `shared` positions in `chunks` pieces of `chunk`
};

struct Words {
  uint32_t w[4];
};

__device__ __forceinline__ Words philox(unsigned long long block, unsigned long long offset, unsigned long long seed) {
  uint32_t c0 = static_cast<uint32_t>(block), c1 = static_cast<uint32_t>(block >> 32);
  uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long a = static_cast<unsigned long long>(0xD2511F53u) * c0, b = static_cast<unsigned long long>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Bit i: element e + i of the mask is kept, i < V.
template <int V>
__device__ __forceinline__ uint32_t kept_bits(const DropParams& p, unsigned long long seed, unsigned long long offset, long long e) {
  uint32_t bits = 0;
  if constexpr (V == 1) {
    const Words r = philox(static_cast<unsigned long long>(e) >> 2, offset, seed);
    const int at = static_cast<int>(e & 3);
    const uint32_t w = at == 0 ? r.w[0] : at == 1 ? r.w[1] : at == 2 ? r.w[2] : r.w[3];
    bits = (w > p.cut) | p.keep_all;
  } else {
#pragma unroll
    for (int b = 0; b < V / 4; ++b) {
      const Words r = philox((static_cast<unsigned long long>(e) >> 2) + b, offset, seed);
#pragma unroll
      for (int i = 0; i < 4; ++i) bits |= static_cast<uint32_t>((r.w[i] > p.cut) | p.keep_all) << (4 * b + i);
    }
  }
  return bits;
}

// U pieces of V elements, their loads before the first store: out may be x or resid, so the compiler keeps the order it is given.
template <int V, int U, typename TX, typename TR, typename Bits>
__device__ __forceinline__ void apply(const TX* x, const TR* resid, TR* out, const long long (&at)[U], const bool (&live)[U], float scale, Bits bits) {
  float v[U][V], r[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (live[u]) {
      load_vec<V>(x + at[u], v[u]);
      if (resid != nullptr) load_vec<V>(resid + at[u], r[u]);
    }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (live[u]) {
      const uint32_t kept = bits(u);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = (kept >> i & 1) ? v[u][i] * scale : 0.f;      // (a select: an infinity or NaN that is dropped leaves no trace)
        v[u][i] = resid != nullptr ? r[u][i] + t : t;
      }
      store_vec<V>(out + at[u], v[u]);
    }
}

__device__ __forceinline__ void stream_of(const DropParams& p, unsigned long long& seed, unsigned long long& offset) {
  seed = p.rng != nullptr ? static_cast<unsigned long long>(p.rng[0]) : p.seed;
  offset = p.rng != nullptr ? static_cast<unsigned long long>(p.rng[1]) : p.offset;
}

// Every element by itself: `inner` of them, a multiple of V.
template <typename TX, typename TR, int V>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const TX* x, const TR* resid, TR* out, const DropParams p) {
  constexpr int U = 2;
  grid_dependency_enter();
  unsigned long long seed, offset;
  stream_of(p, seed, offset);
  constexpr long long kBlock = static_cast<long long>(kThreads) * U * V;
  for (long long base = blockIdx.x * kBlock; base < p.inner; base += gridDim.x * kBlock) {
    long long at[U];
    bool live[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = base + (u * kThreads + static_cast<int>(threadIdx.x)) * V;
      live[u] = at[u] < p.inner;
    }
    apply<V, U>(x, resid, out, at, live, p.scale, [&](int u) { return kept_bits<V>(p, seed, offset, at[u]); });
  }
}

// A shared mask: a thread has V elements of it and the positions of its piece of the shared axis.
template <typename TX, typename TR, int V>
__global__ void __launch_bounds__(kThreads) dropout_shared_kernel(const TX* x, const TR* resid, TR* out, const DropParams p) {
  constexpr int U = 4;
  grid_dependency_enter();
  unsigned long long seed, offset;
  stream_of(p, seed, offset);
  const long long pieces = p.inner / V, total = p.outer * p.chunks * pieces;
  for (long long t = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; t < total; t += static_cast<long long>(gridDim.x) * kThreads) {
    const long long i = t % pieces * V, rest = t / pieces, o = rest / p.chunks, s0 = rest % p.chunks * p.chunk;
    const long long s1 = s0 + p.chunk < p.shared ? s0 + p.chunk : p.shared;
    const uint32_t kept = kept_bits<V>(p, seed, offset, o * p.inner + i);
    for (long long s = s0; s < s1; s += U) {
      long long at[U];
      bool live[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        at[u] = (o * p.shared + s + u) * p.inner + i;
        live[u] = s + u < s1;
      }
      apply<V, U>(x, resid, out, at, live, p.scale, [&](int) { return kept; });
    }
  }
}

template <typename TX, typename TR, int V>
int launch(cudaStream_t stream, const void* x, const void* resid, void* out, DropParams p) {
  const long long sms = sm_count();
  LaunchScope scope(stream, "dropout");
  if (p.shared == 1) {
    p.inner *= p.outer;
    const long long blocks = (p.inner + 2ll * V * kThreads - 1) / (2ll * V * kThreads);
    return launch_kernel(stream, dropout_kernel<TX, TR, V>, static_cast<unsigned>(blocks < sms * 64 ? blocks : sms * 64), kThreads, 0,
                         static_cast<const TX*>(x), static_cast<const TR*>(resid), static_cast<TR*>(out), p);
  }
  // pieces of the shared axis: as long as the device stays full (8 blocks of 256 threads an SM)
  const long long items = p.outer * (p.inner / V), full = sms * 8 * kThreads;
  long long chunks = items >= full ? 1 : (full + items - 1) / items;
  if (chunks > p.shared) chunks = p.shared;
  p.chunk = (p.shared + chunks - 1) / chunks;
  p.chunks = (p.shared + p.chunk - 1) / p.chunk;
  const long long blocks = (items * p.chunks + kThreads - 1) / kThreads;
  return launch_kernel(stream, dropout_shared_kernel<TX, TR, V>, static_cast<unsigned>(blocks < sms * 64 ? blocks : sms * 64), kThreads, 0,
                       static_cast<const TX*>(x), static_cast<const TR*>(resid), static_cast<TR*>(out), p);
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
  d.seed = static_cast<unsigned long long>(seed);
  d.offset = static_cast<unsigned long long>(offset);
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
