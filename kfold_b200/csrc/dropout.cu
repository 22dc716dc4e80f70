// Dropout whose mask is computed from a counter and never stored:  out = (residual +) (kept ? scale x : 0), scale = 1 / (1 - p).  The backward pass is the same
// call on the gradient.
//
// Random words: Philox-4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011),
// key = seed, counter = (e / 4, offset), element e of the mask takes word e % 4 and is dropped when the word is below p 2^32.  So the mask hangs
// on (seed, offset, element) alone: not on the launch shape, the type, or where the tensor lies.
//
// What bounds it: HBM, but the generator is close where every element draws.  Ten rounds are 20 wide multiplications and 20 three-way xors for four words,
// and the integer pipe, which has the xors and the comparisons, is the busiest: what else it had to do was taken from it (an element is added by an instruction
// that runs or does not, instead of by a mask; 32-bit arithmetic inside a block).  384 x 384 x 256 bf16 elements: 35 us with residual, 226 MB at 6.5 TB/s
// (a copy's rate), and 31.5 without, where HBM takes 23; they were 41.5 and 39.3 with masks.  (The comparison as a multiply-add: 90 us the two; wide
// multiply-adds run at half the rate.)
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

// The second round's product that hangs on the block's upper half.
struct Second {
  uint32_t hi, lo;
};
__device__ __forceinline__ Second second_of(uint32_t upper, const Stream& s) {
  if (upper == 0) return {s.a2_hi, s.a2_lo};
  const unsigned long long a2 = static_cast<unsigned long long>(kM0) * (s.b1_hi ^ upper ^ s.key[0]);
  return {static_cast<uint32_t>(a2 >> 32), static_cast<uint32_t>(a2)};
}
// The words of the block with this lower half.
__device__ __forceinline__ Words philox(uint32_t lower, const Second& second, const Stream& s) {
  // the first two rounds
  const unsigned long long a1 = static_cast<unsigned long long>(kM0) * lower;
  const uint32_t d2 = static_cast<uint32_t>(a1 >> 32) ^ s.offset_hi ^ s.key[1], d3 = static_cast<uint32_t>(a1);
  const unsigned long long b2 = static_cast<unsigned long long>(kM1) * d2;
  uint32_t c0 = static_cast<uint32_t>(b2 >> 32) ^ s.b1_lo ^ s.key[2], c1 = static_cast<uint32_t>(b2);
  uint32_t c2 = second.hi ^ d3 ^ s.key[3], c3 = second.lo;
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
  uint32_t cut;                     // kept: word >= cut
  float scale;
  long long outer, shared, inner;   // x is [outer][shared][inner], the mask [outer][inner]
  long long chunks, chunk;          // `shared` positions in `chunks` pieces of `chunk`
};

// V elements as they lie in memory.
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

// The words of V elements from number `at` of block `lower` on: V / 4 blocks, or the one word of V = 1.
template <int V>
__device__ __forceinline__ void words(uint32_t lower, int at, const Second& second, const Stream& stream, uint32_t (&w)[V]) {
  if constexpr (V == 1) {
    const Words r = philox(lower, second, stream);
    w[0] = at == 0 ? r.w[0] : at == 1 ? r.w[1] : at == 2 ? r.w[2] : r.w[3];
  } else {
#pragma unroll
    for (int b = 0; b < V / 4; ++b) {
      const Words r = philox(lower + b, second, stream);      // (V elements start at a multiple of V: no carry into the upper half)
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * b + i] = r.w[i];
    }
  }
}

// sum + (kept ? scale x : 0) and kept ? scale x : 0, as an instruction that runs or does not: no select, and an element that is dropped leaves nothing
// behind whatever it was, an infinity or NaN too.
__device__ __forceinline__ float add_kept(float sum, uint32_t word, uint32_t cut, float x, float scale) {
  asm("{\n\t.reg .pred k;\n\tsetp.ge.u32 k, %1, %2;\n\t@k fma.rn.f32 %0, %3, %4, %0;\n\t}" : "+f"(sum) : "r"(word), "r"(cut), "f"(x), "f"(scale));
  return sum;
}
__device__ __forceinline__ float kept(uint32_t word, uint32_t cut, float x, float scale) {
  float f = 0.f;
  asm("{\n\t.reg .pred k;\n\tsetp.ge.u32 k, %1, %2;\n\t@k mul.rn.f32 %0, %3, %4;\n\t}" : "+f"(f) : "r"(word), "r"(cut), "f"(x), "f"(scale));
  return f;
}

// The words of a mask that serves many elements, as words to and x with as it lies in memory: one instruction for two bf16 elements.
template <typename TX, int V>
__device__ __forceinline__ void mask_of(const uint32_t (&w)[V], uint32_t cut, Piece<TX, V>& m) {
#pragma unroll
  for (int i = 0; i < Piece<TX, V>::kWords; ++i) m.w[i] = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if constexpr (sizeof(TX) == 4) m.w[i] = w[i] >= cut ? 0xffffffffu : 0u;
    else m.w[i / 2] |= w[i] >= cut ? (i & 1 ? 0xffff0000u : 0xffffu) : 0u;
  }
}

constexpr int kBlocksPerSm = 4;
// Pieces at a time where every element draws, and the blocks (an SM) that walk them at most.  384 x 384 x 256 bf16: with residual 2 pieces 36.0 us by up to 64 blocks, 34.6 by
// 24, 38 by 4 pieces; without 34.2 by 2 pieces, 31.5 by 4 and 64 blocks; float32 of 29.6 million elements without 39.8 and 36.2 (37.4 by 16 blocks).
constexpr int pieces_of(bool resid) { return resid ? 2 : 4; }
constexpr int blocks_of(bool resid) { return resid ? 24 : 64; }

// Every element by itself: `inner` of them.  U pieces at a time, their loads before the first store: out may be x or resid, so the
// compiler keeps the order it is given.  A block's elements have the upper half of their counter in common, and all but the last block have every piece:
// what is left for each element is 32-bit arithmetic.  The elements behind the last whole piece, fewer than V, are taken one a thread.  (37.7 million
// bf16 elements and one more: 33.4 us as without it, 37.5 with residual; 121 and 136 where every element of such a count was taken by itself, with a
// block of the generator each.)
template <typename TX, typename TR, int V, bool RESID, bool STATE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) dropout_kernel(const TX* x, const TR* resid, TR* out, const DropParams p) {
  constexpr int U = pieces_of(RESID), kBlock = kThreads * U * V;
  grid_dependency_enter();
  Stream own;
  if (STATE) make_stream(static_cast<unsigned long long>(p.rng[0]), static_cast<unsigned long long>(p.rng[1]), own);
  const Stream& stream = STATE ? own : p.stream;
  const int first = static_cast<int>(threadIdx.x) * V;
  for (long long base = static_cast<long long>(blockIdx.x) * kBlock; base < p.inner; base += static_cast<long long>(gridDim.x) * kBlock) {
    const Second second = second_of(static_cast<uint32_t>(base >> 34), stream);
    const uint32_t lower = static_cast<uint32_t>(base >> 2);
    const int left = static_cast<int>(p.inner - base < kBlock ? p.inner - base : kBlock);
    const TX* xb = x + base;
    const TR* rb = RESID ? resid + base : nullptr;
    TR* ob = out + base;
    auto pieces = [&](auto whole) {
      Piece<TX, V> v[U];
      Piece<TR, V> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = u * kThreads * V + first;
        if (whole || at + V <= left) {
          load_piece<TX, V>(xb + at, v[u]);
          if (RESID) load_piece<TR, V>(rb + at, r[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = u * kThreads * V + first;
        if (whole || at + V <= left) {
          uint32_t w[V];
          words<V>(lower + (static_cast<uint32_t>(at) >> 2), at & 3, second, stream, w);
          float f[V], o[V];
          values<TX, V>(v[u], f);
          if (RESID) values<TR, V>(r[u], o);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = RESID ? add_kept(o[i], w[i], p.cut, f[i], p.scale) : kept(w[i], p.cut, f[i], p.scale);
          store_vec<V>(ob + at, o);
        }
      }
    };
    if (left == kBlock) {
      pieces(std::true_type());
    } else {
      pieces(std::false_type());
      if (V > 1 && static_cast<int>(threadIdx.x) < left % V) {
        const int at = left / V * V + static_cast<int>(threadIdx.x);
        Piece<TX, 1> v;
        Piece<TR, 1> r;
        load_piece<TX, 1>(xb + at, v);
        if (RESID) load_piece<TR, 1>(rb + at, r);
        uint32_t w[1];
        words<1>(lower + (static_cast<uint32_t>(at) >> 2), at & 3, second, stream, w);
        float f[1], o[1];
        values<TX, 1>(v, f);
        if (RESID) values<TR, 1>(r, o);
        o[0] = RESID ? add_kept(o[0], w[0], p.cut, f[0], p.scale) : kept(w[0], p.cut, f[0], p.scale);
        store_vec<1>(ob + at, o);
      }
    }
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
    uint32_t w[V];
    const unsigned long long e = static_cast<unsigned long long>(o * p.inner + i);
    words<V>(static_cast<uint32_t>(e >> 2), static_cast<int>(e & 3), second_of(static_cast<uint32_t>(e >> 34), stream), stream, w);
    Piece<TX, V> m;
    mask_of<TX, V>(w, p.cut, m);
    const long long first = (o * p.shared + s0) * p.inner + i;
    const TX* xs = x + first;
    const TR* rs = RESID ? resid + first : nullptr;
    TR* os = out + first;
    for (; left > 0; left -= U) {
      Piece<TX, V> v[U];
      Piece<TR, V> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) {
          load_piece<TX, V>(xs + u * p.inner, v[u]);
          if (RESID) load_piece<TR, V>(rs + u * p.inner, r[u]);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) {
#pragma unroll
          for (int k = 0; k < Piece<TX, V>::kWords; ++k) v[u].w[k] &= m.w[k];
          float f[V], add[V];
          values<TX, V>(v[u], f);
          if (RESID) values<TR, V>(r[u], add);
#pragma unroll
          for (int k = 0; k < V; ++k) f[k] = RESID ? fmaf(f[k], p.scale, add[k]) : f[k] * p.scale;
          store_vec<V>(os + u * p.inner, f);
        }
      xs += U * p.inner;
      if (RESID) rs += U * p.inner;
      os += U * p.inner;
    }
  }
}

template <typename TX, typename TR, int V, bool RESID, bool STATE>
int launch_each(cudaStream_t stream, const void* x, const void* resid, void* out, DropParams p) {
  p.inner *= p.outer;
  constexpr long long kBlock = static_cast<long long>(pieces_of(RESID)) * V * kThreads;
  const long long blocks = (p.inner + kBlock - 1) / kBlock, most = static_cast<long long>(sm_count()) * blocks_of(RESID);
  LaunchScope scope(stream, "dropout");
  return launch_kernel(stream, dropout_kernel<TX, TR, V, RESID, STATE>, static_cast<unsigned>(blocks < most ? blocks : most), kThreads, 0,
                       static_cast<const TX*>(x), static_cast<const TR*>(resid), static_cast<TR*>(out), p);
}
template <typename TX, typename TR, int V, bool RESID, bool STATE>
int launch_shared(cudaStream_t stream, const void* x, const void* resid, void* out, DropParams p) {
  // pieces of the shared axis: as many as fill the device once
  const long long sms = sm_count(), items = p.outer * (p.inner / V), full = sms * kBlocksPerSm * kThreads;
  long long chunks = items >= full ? 1 : full / items;
  if (chunks > p.shared) chunks = p.shared;
  p.chunk = (p.shared + chunks - 1) / chunks;
  p.chunks = (p.shared + p.chunk - 1) / p.chunk;
  const long long blocks = (items * p.chunks + kThreads - 1) / kThreads;
  LaunchScope scope(stream, "dropout");
  return launch_kernel(stream, dropout_shared_kernel<TX, TR, V, RESID, STATE>, static_cast<unsigned>(blocks < sms * 64 ? blocks : sms * 64), kThreads, 0,
                       static_cast<const TX*>(x), static_cast<const TR*>(resid), static_cast<TR*>(out), p);
}
template <typename TX, typename TR, int V, bool SHARED>
int launch(cudaStream_t stream, const void* x, const void* resid, void* out, const DropParams& p) {
  auto by = [&](auto has_resid, auto state) {
    if constexpr (SHARED) return launch_shared<TX, TR, V, has_resid.value, state.value>(stream, x, resid, out, p);
    else return launch_each<TX, TR, V, has_resid.value, state.value>(stream, x, resid, out, p);
  };
  const std::true_type yes;
  const std::false_type no;
  if (resid != nullptr) return p.rng != nullptr ? by(yes, yes) : by(yes, no);
  return p.rng != nullptr ? by(no, yes) : by(no, no);
}

template <typename TX, typename TR>
int dispatch(cudaStream_t stream, const void* x, const void* resid, void* out, const DropParams& p) {
  constexpr int V = std::is_same<TX, __nv_bfloat16>::value && std::is_same<TR, __nv_bfloat16>::value ? 8 : 4;
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(resid) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (p.shared == 1) return aligned ? launch<TX, TR, V, false>(stream, x, resid, out, p) : launch<TX, TR, 1, false>(stream, x, resid, out, p);
  // (neighbours in memory whose mask elements are neighbours: a run of the inner axis)
  if (aligned && p.inner % V == 0) return launch<TX, TR, V, true>(stream, x, resid, out, p);
  if (aligned && p.inner % 4 == 0) return launch<TX, TR, 4, true>(stream, x, resid, out, p);
  return launch<TX, TR, 1, true>(stream, x, resid, out, p);
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
  cudaStream_t s = as_stream(stream);
  if (drop_below == 1ll << 32) {        // nothing is kept: the kernels' comparison has no word for it
    const size_t bytes = static_cast<size_t>(outer) * shared * inner * (out_dtype == KFB_FP32 ? 4 : 2);
    if (residual == nullptr) KFB_CUDA(cudaMemsetAsync(out, 0, bytes, s));
    else if (residual != out) KFB_CUDA(cudaMemcpyAsync(out, residual, bytes, cudaMemcpyDeviceToDevice, s));
    return KFB_OK;
  }
  DropParams d = {};
  d.rng = rng;
  make_stream(static_cast<unsigned long long>(seed), static_cast<unsigned long long>(offset), d.stream);
  d.cut = static_cast<uint32_t>(drop_below);
  d.scale = scale;
  d.outer = outer;
  d.shared = shared;
  d.inner = inner;
  if (x_dtype == KFB_BF16)
    return out_dtype == KFB_BF16 ? dispatch<__nv_bfloat16, __nv_bfloat16>(s, x, residual, out, d) : dispatch<__nv_bfloat16, float>(s, x, residual, out, d);
  return dispatch<float, float>(s, x, residual, out, d);
}
