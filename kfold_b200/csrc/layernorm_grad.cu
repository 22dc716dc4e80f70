// The gradient of LayerNorm.  With m, r the row's mean and 1 / sqrt(var + eps), z = (x - m) r and g = w dy:
//   dx = r (g - mean(g) - z mean(g z)),   dw = sum over rows of dy z,   db = sum over rows of dy.
//
// What bounds it: x and dy in, dx out, and nothing else is large, so HBM.  The statistics are taken again from the row, which is in registers
// anyway, instead of being saved by the forward pass (8 bytes a row and two more tensors for the caller to keep).
// Split: a row is held by 8, 16 or 32 lanes, in 16-byte pieces where the width allows; a warp has enough rows in flight to cover the memory's
// latency, keeps its lanes' shares of dw and db in registers from row to row, and a block leaves one row of partial sums.  A second kernel adds
// those in the blocks' order, so that the result does not hang on which block was first: no atomics.
//
// Measured (graph replays): 147 456 rows of 256 bf16 channels 43 us, of which dx is 39, 226 MB at 5.8 TB/s (a copy has 6.5), and the sums over the blocks
// 4; 63 001 rows of 128 13.6 and 9.5; 301 rows of 384 float32 4.9, 64 4.2 in one launch.  The next rows' loads have to stand before this step's stores, and the row
// sums of a step be interleaved: 74 us where the first is 43 without.  49 152 rows of 505 channels 83 -> 44 us.
#include <cuda_bf16.h>

#include <mutex>
#include <type_traits>

#include "ops_common.cuh"
#include "ptx.cuh"
#include "vec_io.cuh"

namespace kfb {
namespace {

constexpr int kWarps = 8;

// V elements as they lie in memory: what is on its way takes no more registers than its bytes.
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T)), kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p, bool there) {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 t = there ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0, 0, 0, 0);
        w[4 * i] = t.x;
        w[4 * i + 1] = t.y;
        w[4 * i + 2] = t.z;
        w[4 * i + 3] = t.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 t = there ? *reinterpret_cast<const uint2*>(p) : make_uint2(0, 0);
      w[0] = t.x;
      w[1] = t.y;
    } else if constexpr (kBytes == 4) {
      w[0] = there ? *reinterpret_cast<const uint32_t*>(p) : 0u;
    } else {
      w[0] = there ? *reinterpret_cast<const unsigned short*>(p) : 0u;
    }
  }
  __device__ __forceinline__ void values(float* v) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
      else v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
  }
};

enum Params : int { kNone = 0, kPartial = 1, kCluster = 2 };   // dw, db: not wanted; a row of partial sums a block; the whole grid is one cluster

// A float of the shared memory of the cluster's CTA `rank`, at the place of this CTA's `p`.
__device__ __forceinline__ float peer_float(const float* p, unsigned rank) {
  float v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(ptx::smem_u32(p)), "r"(rank) : "memory");
  return v;
}

// LANES lanes hold a row, P pieces of V channels each; R rows in flight for each group of lanes.  EXACT: c == LANES * V * P.
template <typename TX, typename TD, int V, int LANES, int P, int R, bool EXACT, int MODE>
__global__ void __launch_bounds__(32 * kWarps) layernorm_grad_kernel(const TD* dy, const TX* x, const float* w, TX* dx, float* partial, float* dw,
                                                                     float* db, long long rows, int c, float eps) {
  constexpr bool PARAMS = MODE != kNone;
  constexpr int N = P * V, kGroups = 32 / LANES, kRows = kGroups * R;
  grid_dependency_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % LANES;
  const float inv_c = 1.0f / static_cast<float>(c);
  auto channel = [&](int p) { return (p * LANES + sub) * V; };
  auto inside = [&](int p) { return EXACT || channel(p) < c; };
  float wv[N], aw[PARAMS ? N : 1], ab[PARAMS ? N : 1];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < V; ++i) wv[p * V + i] = w != nullptr && inside(p) ? w[channel(p) + i] : 1.0f;
#pragma unroll
  for (int i = 0; i < (PARAMS ? N : 1); ++i) aw[i] = ab[i] = 0.f;

  // The next rows' pieces are on their way while these are worked on.  (They have to be asked for before this step's stores: behind one, a load waits.)
  const long long step = static_cast<long long>(gridDim.x) * kWarps * kRows;
  Raw<TX, V> x_raw[R][P];
  Raw<TD, V> d_raw[R][P];
  auto fetch = [&](long long base) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * kGroups + lane / LANES;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const bool there = row < rows && inside(p);
        x_raw[r][p].load(x + row * c + channel(p), there);
        d_raw[r][p].load(dy + row * c + channel(p), there);
      }
    }
  };
  long long base = (static_cast<long long>(blockIdx.x) * kWarps + warp) * kRows;
  if (base < rows) fetch(base);
  for (; base < rows; base += step) {
    float xv[R][N], dv[R][N], mean[R], sg[R], q[R], sz[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        x_raw[r][p].values(&xv[r][p * V]);
        d_raw[r][p].values(&dv[r][p * V]);
      }
    if (base + step < rows) fetch(base + step);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = sg[r] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        mean[r] += xv[r][i];
        sg[r] = fmaf(dv[r][i], wv[i], sg[r]);
      }
    }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        mean[r] += __shfl_xor_sync(0xffffffffu, mean[r], m);
        sg[r] += __shfl_xor_sync(0xffffffffu, sg[r], m);
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] *= inv_c;
      q[r] = sz[r] = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = p * V; i < p * V + V; ++i) {
          xv[r][i] = inside(p) ? xv[r][i] - mean[r] : 0.f;
          q[r] = fmaf(xv[r][i], xv[r][i], q[r]);
          sz[r] = fmaf(dv[r][i] * wv[i], xv[r][i], sz[r]);
        }
    }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        q[r] += __shfl_xor_sync(0xffffffffu, q[r], m);
        sz[r] += __shfl_xor_sync(0xffffffffu, sz[r], m);
      }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = base + r * kGroups + lane / LANES;
      if (row >= rows) continue;
      const float rstd = rsqrtf(q[r] * inv_c + eps);
      sz[r] *= inv_c * rstd;
      sg[r] *= inv_c;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float z = xv[r][p * V + i] * rstd, d = dv[r][p * V + i];
          o[i] = rstd * (fmaf(d, wv[p * V + i], -sg[r]) - z * sz[r]);
          if constexpr (PARAMS) {
            aw[p * V + i] = fmaf(d, z, aw[p * V + i]);
            ab[p * V + i] += d;
          }
        }
        if (inside(p)) store_vec<V>(dx + row * c + channel(p), o);
      }
    }
  }

  if constexpr (PARAMS) {
    __shared__ float s_sum[kWarps][LANES * N];
    __shared__ float s_total[MODE == kCluster ? 2 * LANES * N : 1];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float(&a)[N] = which ? ab : aw;
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int m = LANES; m < 32; m <<= 1) a[i] += __shfl_xor_sync(0xffffffffu, a[i], m);
      }
      if (lane < LANES) {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < V; ++i) s_sum[warp][channel(p) + i] = a[p * V + i];
      }
      __syncthreads();
      for (int ch = threadIdx.x; ch < c; ch += 32 * kWarps) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) t += s_sum[k][ch];
        if constexpr (MODE == kCluster) s_total[which * c + ch] = t;
        else partial[(static_cast<long long>(blockIdx.x) * 2 + which) * c + ch] = t;
      }
      __syncthreads();
    }
    if constexpr (MODE == kCluster) {
      // the blocks' sums, in their order, from one another's shared memory: few rows then take one launch
      ptx::cluster_sync();
      for (int i = blockIdx.x * 32 * kWarps + threadIdx.x; i < 2 * c; i += gridDim.x * 32 * kWarps) {
        float t = 0.f;
        for (unsigned b = 0; b < gridDim.x; ++b) t += peer_float(&s_total[i], b);
        float* d = i < c ? dw : db;
        if (d != nullptr) d[i < c ? i : i - c] = t;
      }
      ptx::cluster_sync();
    }
  }
}

// dw and db (either may be null) from the blocks' partial sums, in the order of the blocks.  A block takes 32 channels of the 2 c.
__global__ void __launch_bounds__(1024) layernorm_grad_sum_kernel(const float* partial, float* dw, float* db, int blocks, int c) {
  __shared__ float s[32][33];
  grid_dependency_enter();
  const int col = blockIdx.x * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  float t = 0.f;
  if (col < 2 * c) {
#pragma unroll 4
    for (int b = part; b < blocks; b += 32) t += partial[static_cast<long long>(b) * 2 * c + col];
  }
  s[part][threadIdx.x % 32] = t;
  __syncthreads();
  if (part == 0 && col < 2 * c) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += s[k][threadIdx.x];
    if (col < c) {
      if (dw != nullptr) dw[col] = t;
    } else if (db != nullptr) {
      db[col - c] = t;
    }
  }
}

constexpr int kBlocksPerSm = 8;      // at most: the workspace's partial sums are sized by it
constexpr int kMostSms = 160;
constexpr int kMostCluster = 8;      // blocks of a cluster.  Up to four steps of each of them they are faster than many blocks and a second launch

struct Args {
  cudaStream_t stream;
  const void *dy, *x;
  const float* w;
  void* dx;
  float *dw, *db, *partial;
  long long rows;
  int c;
  float eps;
};

template <typename TX, typename TD, int V, int LANES, int P, bool EXACT, int MODE>
int launch_mode(const Args& a) {
  constexpr int N = V * P, R = N <= 8 ? 2 : 1;
  auto kernel = layernorm_grad_kernel<TX, TD, V, LANES, P, R, EXACT, MODE>;
  const long long step = static_cast<long long>(kWarps) * (32 / LANES) * R, want = (a.rows + step - 1) / step;
  if constexpr (MODE == kPartial) {
    if (want <= 4 * kMostCluster) return launch_mode<TX, TD, V, LANES, P, EXACT, kCluster>(a);
  }
  int blocks = static_cast<int>(want < kMostCluster ? want : kMostCluster);
  if constexpr (MODE != kCluster) {
    static std::once_flag once;
    static int held = 1;
    std::call_once(once, [&] {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, 32 * kWarps, 0) != cudaSuccess) cudaGetLastError();
      held = held < 1 ? 1 : held > kBlocksPerSm ? kBlocksPerSm : held;
    });
    const long long sms = sm_count() < kMostSms ? sm_count() : kMostSms;
    blocks = static_cast<int>(want < sms * held ? want : sms * held);
  }
  {
    LaunchScope scope(a.stream, "layernorm_grad");
    KFB_TRY(launch_kernel_clustered(a.stream, kernel, MODE == kCluster ? blocks : 1, blocks, 32 * kWarps, 0, static_cast<const TD*>(a.dy),
                                    static_cast<const TX*>(a.x), a.w, static_cast<TX*>(a.dx), a.partial, a.dw, a.db, a.rows, a.c, a.eps));
  }
  if (MODE == kPartial) {
    LaunchScope scope(a.stream, "layernorm_grad_sum");
    KFB_TRY(launch_kernel(a.stream, layernorm_grad_sum_kernel, cdiv(2 * a.c, 32), 1024, 0, const_cast<const float*>(a.partial), a.dw, a.db, blocks,
                          a.c));
  }
  return KFB_OK;
}

template <typename TX, typename TD, int V, int LANES, int P, bool EXACT>
int launch(const Args& a) {
  return a.dw != nullptr || a.db != nullptr ? launch_mode<TX, TD, V, LANES, P, EXACT, kPartial>(a) : launch_mode<TX, TD, V, LANES, P, EXACT, kNone>(a);
}

template <typename TX, typename TD>
int dispatch(const Args& a) {
  constexpr bool kHalf = std::is_same<TX, __nv_bfloat16>::value && std::is_same<TD, __nv_bfloat16>::value;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.dx);
  if ((at & 15) == 0) {
    if constexpr (kHalf) {
      switch (a.c) {
        case 64: return launch<TX, TD, 8, 8, 1, true>(a);
        case 128: return launch<TX, TD, 8, 16, 1, true>(a);
        case 256: return launch<TX, TD, 8, 32, 1, true>(a);
        case 384: return launch<TX, TD, 8, 16, 3, true>(a);
        case 768: return launch<TX, TD, 8, 32, 3, true>(a);
      }
    } else {
      switch (a.c) {
        case 64: return launch<TX, TD, 4, 16, 1, true>(a);
        case 128: return launch<TX, TD, 4, 32, 1, true>(a);
        case 256: return launch<TX, TD, 4, 32, 2, true>(a);
        case 384: return launch<TX, TD, 4, 32, 3, true>(a);
        case 768: return launch<TX, TD, 4, 32, 6, true>(a);
      }
    }
    if (a.c % 4 == 0) {
      if (a.c <= 256) return launch<TX, TD, 4, 32, 2, false>(a);
      if (a.c <= 512) return launch<TX, TD, 4, 32, 4, false>(a);
      return launch<TX, TD, 4, 32, 8, false>(a);
    }
  }
  if (a.c <= 256) return launch<TX, TD, 1, 32, 8, false>(a);
  if (a.c <= 512) return launch<TX, TD, 1, 32, 16, false>(a);
  return launch<TX, TD, 1, 32, 32, false>(a);
}

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API size_t kfb_layernorm_bwd_workspace_bytes(int c) {
  return align_up(static_cast<size_t>(kMostSms) * kBlocksPerSm * 2 * (c > 0 ? c : 0) * sizeof(float), 256);
}

KFB_API int kfb_layernorm_bwd(const void* dy, const void* x, const float* weight, void* dx, float* dweight, float* dbias, void* workspace,
                              size_t workspace_bytes, long long rows, int c, float eps, int dy_dtype, int x_dtype, void* stream) {
  KFB_CHECK_ARG(rows >= 0 && c > 0, "layernorm_bwd: rows %lld, channels %d", rows, c);
  if (c > 1024) {
    set_error("layernorm_bwd: channel count %d above 1024 is not supported", c);
    return KFB_ERR_UNSUPPORTED;
  }
  const bool params = dweight != nullptr || dbias != nullptr;
  KFB_CHECK_ARG((dy_dtype == KFB_BF16 || dy_dtype == KFB_FP32) && (x_dtype == KFB_BF16 || x_dtype == KFB_FP32), "layernorm_bwd: bad dtype %d / %d",
                dy_dtype, x_dtype);
  cudaStream_t s = as_stream(stream);
  if (rows == 0) {
    if (dweight != nullptr) KFB_CUDA(cudaMemsetAsync(dweight, 0, static_cast<size_t>(c) * 4, s));
    if (dbias != nullptr) KFB_CUDA(cudaMemsetAsync(dbias, 0, static_cast<size_t>(c) * 4, s));
    return KFB_OK;
  }
  KFB_CHECK_ARG(dy != nullptr && x != nullptr && dx != nullptr, "layernorm_bwd: null tensor");
  KFB_CHECK_ARG(!params || (workspace != nullptr && workspace_bytes >= kfb_layernorm_bwd_workspace_bytes(c)),
                "layernorm_bwd: workspace %zu < %zu bytes", workspace_bytes, kfb_layernorm_bwd_workspace_bytes(c));
  KFB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "layernorm_bwd: workspace must be 256-byte aligned");
  const Args a = {s, dy, x, weight, dx, dweight, dbias, static_cast<float*>(workspace), rows, c, eps};
  if (x_dtype == KFB_BF16)
    return dy_dtype == KFB_BF16 ? dispatch<__nv_bfloat16, __nv_bfloat16>(a) : dispatch<__nv_bfloat16, float>(a);
  return dy_dtype == KFB_BF16 ? dispatch<float, __nv_bfloat16>(a) : dispatch<float, float>(a);
}

}  // extern "C"
