// Rows put away in 8 bits and taken back (the format is in row_teams.cuh).
//
// What bounds it: HBM, 2 or 4 bytes a value one way and 33 / 32 the other.  A lane takes eight neighbouring channels of a row where they are a multiple of eight and lie
// on 16-byte boundaries, four lanes then hold a group of 32.  Rows of whole groups have no ends: their pieces are
// numbered through, and a thread has four of them on their way: 147 456 rows of 256 bf16 channels 20 us, 18 us back, 5.8 and 6.4 TB/s.
#include "ops_common.cuh"
#include "row_teams.cuh"

namespace kfb {
namespace {

// Rows of `groups` groups of 32.  VEC: four pieces of eight neighbouring channels a group, numbered through.  Otherwise, taken back: pieces of eight groups, a warp's, a lane
// has every 32nd channel.
template <bool VEC>
__device__ __forceinline__ long long pieces_of_row(int groups) { return VEC ? 4ll * groups : (groups + kPiece - 1) / kPiece * 32ll; }
// (first channel of a lane's piece number i of a row)
template <bool VEC>
__device__ __forceinline__ int first_channel(int i) { return VEC ? i * kPiece : i / 32 * (32 * kPiece) + i % 32; }

// Eight neighbouring channels, of which n are there, one by one.  (What a lane asks for lies in one or two sectors, which come once; a group's largest magnitude is then
// two exchanges between lanes, where a group spread over a warp takes a reduction for every channel: 300 000 rows of 100 bf16 channels 43 us and 99.)
template <typename T>
__device__ __forceinline__ Pairs load_near(const T* p, int n) {
  float f[kPiece];
#pragma unroll
  for (int i = 0; i < kPiece; ++i) f[i] = i < n ? static_cast<float>(p[i]) : 0.f;
  return of_floats(f);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) compress_kernel(const T* x, uint8_t* q, uint8_t* e, long long pieces, int c, int groups) {
  grid_dependency_enter();
  const long long per_row = 4ll * groups;
  // (a warp's lanes leave the loop together: pieces beyond the end have no values)
  for (long long first = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x / 32 * 32; first < pieces; first += gridDim.x * 256ll) {
    const long long i = first + threadIdx.x % 32, row = i / per_row;
    const int ch = static_cast<int>(i - row * per_row) * kPiece, n = i < pieces ? min(max(c - ch, 0), kPiece) : 0;
    Pairs v;
    if constexpr (VEC) v = load_piece<T, true>(x + row * c + ch, n);
    else v = load_near(x + row * c + ch, n);
    const uint32_t ex = exponent8(group_top(top_of(v)));
    const uint2 b = bytes8(v, ex);
    uint8_t* to = q + row * c + ch;
    if constexpr (VEC) {
      if (n > 0) *reinterpret_cast<uint2*>(to) = b;
    } else {
#pragma unroll
      for (int k = 0; k < kPiece; ++k)
        if (k < n) to[k] = static_cast<uint8_t>((k < 4 ? b.x : b.y) >> 8 * (k & 3));
    }
    if (n > 0 && threadIdx.x % 4 == 0) e[row * groups + ch / kGroup8] = static_cast<uint8_t>(ex);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) expand_kernel(const uint8_t* q, const uint8_t* e, T* x, long long rows, int c, int groups) {
  grid_dependency_enter();
  const long long per_row = pieces_of_row<VEC>(groups), pieces = rows * per_row;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < pieces; i += gridDim.x * 256ll) {
    const long long row = i / per_row;
    const int ch = first_channel<VEC>(static_cast<int>(i - row * per_row)), n = channels_of<VEC>(c, ch);
    store_piece<VEC>(x + row * c + ch, load_piece8<VEC>(q + row * c + ch, e + row * groups + ch / kGroup8, n), n);
  }
}

constexpr int kAhead = 4;
template <typename T>
__global__ void __launch_bounds__(256) compress_whole_kernel(const T* x, uint8_t* q, uint8_t* e, long long pieces) {
  grid_dependency_enter();
  const long long step = 256ll * kAhead;
  for (long long first = blockIdx.x * step; first < pieces; first += gridDim.x * step) {
    Pairs v[kAhead];
    long long i[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      i[k] = first + k * 256 + threadIdx.x;
      v[k] = load_piece<T, true>(x + i[k] * kPiece, i[k] < pieces ? kPiece : 0);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      store_piece8<true>(q + i[k] * kPiece, e + i[k] / 4, v[k], top_of(v[k]), i[k] < pieces ? kPiece : 0, threadIdx.x % 32);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) expand_whole_kernel(const uint8_t* q, const uint8_t* e, T* x, long long pieces) {
  grid_dependency_enter();
  const long long step = 256ll * kAhead;
  for (long long first = blockIdx.x * step; first < pieces; first += gridDim.x * step) {
    uint2 b[kAhead];
    uint32_t ex[kAhead];
    long long i[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      i[k] = first + k * 256 + threadIdx.x;
      const bool there = i[k] < pieces;
      b[k] = there ? *reinterpret_cast<const uint2*>(q + i[k] * kPiece) : make_uint2(0, 0);
      ex[k] = there ? e[i[k] / 4] : 0u;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) store_piece<true>(x + i[k] * kPiece, values8(b[k], ex[k]), i[k] < pieces ? kPiece : 0);
  }
}

template <typename T>
int compress_as(cudaStream_t s, const void* x, void* q, void* e, long long rows, int c) {
  const long long pieces = rows * groups8(c) * 4;
  const bool vec = c % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0, whole = vec && c % kGroup8 == 0;
  const long long block = whole ? 256 * kAhead : 256, want = (pieces + block - 1) / block, most = (whole ? 8ll : 16ll) * sm_count();
  const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
  LaunchScope scope(s, "compress");
  if (whole) return launch_kernel(s, compress_whole_kernel<T>, blocks, 256, 0, static_cast<const T*>(x), static_cast<uint8_t*>(q), static_cast<uint8_t*>(e), pieces);
  return launch_kernel(s, vec ? compress_kernel<T, true> : compress_kernel<T, false>, blocks, 256, 0, static_cast<const T*>(x), static_cast<uint8_t*>(q),
                       static_cast<uint8_t*>(e), pieces, c, groups8(c));
}

template <typename T>
int expand_as(cudaStream_t s, const void* q, const void* e, void* x, long long rows, int c) {
  const long long pieces = rows * groups8(c) * 4;
  const bool vec = c % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0, whole = vec && c % kGroup8 == 0;
  const long long block = whole ? 256 * kAhead : 256, want = (pieces + block - 1) / block, most = (whole ? 8ll : 16ll) * sm_count();
  const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
  LaunchScope scope(s, "expand");
  if (whole) return launch_kernel(s, expand_whole_kernel<T>, blocks, 256, 0, static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(e), static_cast<T*>(x), pieces);
  return launch_kernel(s, vec ? expand_kernel<T, true> : expand_kernel<T, false>, blocks, 256, 0, static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(e),
                       static_cast<T*>(x), rows, c, groups8(c));
}

int check(const char* name, const void* a, const void* b, const void* d, long long rows, int c, int dtype) {
  KFB_CHECK_ARG(rows >= 0 && rows < (1ll << 40) && c > 0 && c <= 65536, "%s: rows %lld, channels %d", name, rows, c);
  KFB_CHECK_ARG(dtype == KFB_BF16 || dtype == KFB_FP32, "%s: bad dtype %d", name, dtype);
  KFB_CHECK_ARG(rows == 0 || (a != nullptr && b != nullptr && d != nullptr), "%s: null tensor", name);
  return KFB_OK;
}

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API int kfb_compress(const void* x, void* values, void* exponents, long long rows, int c, int dtype, void* stream) {
  KFB_TRY(check("compress", x, values, exponents, rows, c, dtype));
  if (rows == 0) return KFB_OK;
  cudaStream_t s = as_stream(stream);
  return dtype == KFB_BF16 ? compress_as<__nv_bfloat16>(s, x, values, exponents, rows, c) : compress_as<float>(s, x, values, exponents, rows, c);
}

KFB_API int kfb_expand(const void* values, const void* exponents, void* x, long long rows, int c, int dtype, void* stream) {
  KFB_TRY(check("expand", x, values, exponents, rows, c, dtype));
  if (rows == 0) return KFB_OK;
  cudaStream_t s = as_stream(stream);
  return dtype == KFB_BF16 ? expand_as<__nv_bfloat16>(s, values, exponents, x, rows, c) : expand_as<float>(s, values, exponents, x, rows, c);
}

}  // extern "C"
