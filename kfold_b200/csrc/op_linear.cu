// A linear layer with its tail, and its gradient (training; inference has kfb_gemm_bf16 and kfb_linear_fp32):
//   z = x W^T + b,  y = f(z) (+ residual);   dz = dy f'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz.
//
// z is computed again where f' needs it: 2 of then 8 operations per row and weight, where keeping it is 2 bytes a row and output.  z stays float32;
// dz is rounded to bf16 once, as an operand, and db is summed before that.
// Rows are taken in pieces, so that the workspace does not grow with them; dW is summed over pieces of rows in float32 planes and added up at the end, in
// an order that depends on the sizes alone.
#include "linear_tail.cuh"
#include "matmul.cuh"
#include "ops_common.cuh"

namespace kfb {
namespace {

constexpr int kTailCols = 256, kTailWarps = 8;       // of a block: a lane has 8 columns of every eighth row

struct TailParams {
  const float* z;              // [rows][n] products, null: none (backward without f: only the sums)
  const float* bias;
  const void *resid, *dy;      // forward: added to f; backward: the gradient
  void* out;                   // forward
  __nv_bfloat16* dz;           // backward: operand of the products, or its three parts `plane` apart (precise)
  long long plane;
  float* partial;              // backward: [row block][n] sums of dz
  long long rows;
  int n, rows_per_block, parts, resid_fp32, out_fp32, dy_fp32;
};

__device__ __forceinline__ void load8f(const void* p, long long o, int fp32, float* v) {
  if (fp32) {
    const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(p) + o)[0], b = reinterpret_cast<const float4*>(static_cast<const float*>(p) + o)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + o);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

template <int ACT, bool BACK>
__global__ void __launch_bounds__(32 * kTailWarps) linear_tail_kernel(const TailParams p) {
  __shared__ float s[kTailWarps][kTailCols];
  grid_dependency_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * kTailCols + lane * 8;
  const bool there = col < p.n;                       // (n is a multiple of 8)
  float bias[8], sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bias[i] = there && p.bias != nullptr ? p.bias[col + i] : 0.f;
    sum[i] = 0.f;
  }
  const long long first = static_cast<long long>(blockIdx.y) * p.rows_per_block;
  const long long end = first + p.rows_per_block < p.rows ? first + p.rows_per_block : p.rows;
  if (there) {
    for (long long r = first + warp; r < end; r += kTailWarps) {
      const long long o = r * p.n + col;
      float z[8], v[8];
      if (p.z != nullptr) {
        load8f(p.z, o, 1, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] += bias[i];
      }
      if constexpr (BACK) {
        load8f(p.dy, o, p.dy_fp32, v);
        if (p.z != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= slope<ACT>(z[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += v[i];
        if (p.dz != nullptr) {
          if (p.parts == 1) {
            *reinterpret_cast<uint4*>(p.dz + o) = pack8(v);
          } else {
            __nv_bfloat16 q[3][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) split3(v[i], q[0][i], q[1][i], q[2][i]);
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(p.dz + k * p.plane + o) = *reinterpret_cast<const uint4*>(q[k]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = activation<ACT>(z[i]);
        if (p.resid != nullptr) {
          load8f(p.resid, o, p.resid_fp32, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) z[i] += v[i];
        }
        if (p.out_fp32) {
          float4* d = reinterpret_cast<float4*>(static_cast<float*>(p.out) + o);
          d[0] = make_float4(z[0], z[1], z[2], z[3]);
          d[1] = make_float4(z[4], z[5], z[6], z[7]);
        } else {
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + o) = pack8(z);
        }
      }
    }
  }
  if constexpr (BACK) {
    if (p.partial == nullptr) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) s[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    const int c = blockIdx.x * kTailCols + threadIdx.x;
    if (c < p.n) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kTailWarps; ++w) t += s[w][threadIdx.x];
      p.partial[static_cast<long long>(blockIdx.y) * p.n + c] = t;
    }
  }
}

// out[c] (+)= sum over rows of partial[row][c], in an order of their number alone.
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* partial, float* out, int rows, int n, int add) {
  __shared__ float s[32][33];
  grid_dependency_enter();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float t = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int b = part; b < rows; b += 32) t += partial[static_cast<long long>(b) * n + col];
  }
  s[part][lane] = t;
  __syncthreads();
  if (part == 0 && col < n) {
    t = add ? out[col] : 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += s[k][lane];
    out[col] = t;
  }
}

constexpr int kMostRowBlocks = 592;

template <bool BACK>
int launch_tail(cudaStream_t stream, TailParams p, int act, int* row_blocks) {
  const int cols = cdiv(p.n, kTailCols);
  long long blocks = kMostRowBlocks / cols;
  if (blocks < 1) blocks = 1;
  long long per = (p.rows + blocks - 1) / blocks;
  if (per < kTailWarps) per = kTailWarps;
  p.rows_per_block = static_cast<int>(per);
  const int rows = static_cast<int>((p.rows + per - 1) / per);
  *row_blocks = rows;
  auto kernel = act == kSigmoid ? linear_tail_kernel<kSigmoid, BACK> : act == kSilu ? linear_tail_kernel<kSilu, BACK>
                : act == kGelu ? linear_tail_kernel<kGelu, BACK> : act == kRelu ? linear_tail_kernel<kRelu, BACK> : linear_tail_kernel<kIdentity, BACK>;
  LaunchScope scope(stream, "linear_tail");
  return launch_kernel(stream, kernel, dim3(cols, rows), 32 * kTailWarps, 0, p);
}

bool widths_ok(int k, int n) { return k > 0 && k % 8 == 0 && n > 0 && n % 8 == 0 && k <= 65536 && n <= 65536; }

// Which kernels a call takes: many bf16 rows those for CTA pairs, which keep nothing but dz; others products into float32 and the tail by itself.
struct Ways {
  bool z, dx, dw;          // the products with what follows them, those for dx, those for dW
};
Ways ways(long long rows, int k, int n, int act, int precise, int wide, int wanted) {
  Ways w = {};
  if (precise) return w;
  w.z = !wide && (wanted == 0 || act != kIdentity) && linear_pair_ok(rows, n, k);
  w.dx = (wanted & 1) && linear_pair_ok(rows, k, n);
  w.dw = (wanted & 2) && linear_weights_ok(n, k);
  return w;
}

// Rows of a piece: as many as keep what a row needs below half a gigabyte.
long long piece_rows(long long rows, int k, int n, int precise, bool z) {
  const long long per_row = 2ll * n + (z ? 4ll * n : 0) + (precise ? 6ll * (k + n) : 0), most = ((1ll << 29) / per_row + 127) / 128 * 128;
  return rows < most ? rows : most;
}

// Blocks of 64 rows that a plane of dW takes from a piece: two tiles an SM.
int blocks_per_plane(long long piece, int k, int n) {
  const long long tiles = static_cast<long long>(cdiv(n, 128)) * cdiv(k, 128), blocks = (piece + 63) / 64, want = 2 * 148 / tiles;
  const long long s = want < 1 ? 1 : want < blocks ? want : blocks;
  return static_cast<int>((blocks + s - 1) / s);
}
// (a shorter last piece has no more planes than a full one)
int weight_splits(long long rows, int per) { return static_cast<int>(((rows + 63) / 64 + per - 1) / per); }

struct Room {
  Ways way;
  long long piece;
  int per_plane, splits;
  float* z;
  __nv_bfloat16 *dz, *x3, *w3;
  float *planes, *partial;
  size_t bytes;
};

// wanted: 0 forward, else a sum of 1 dx, 2 dW, 4 db; wide: the result or its gradient is float32 beside bf16
Room carve(void* base, long long rows, int k, int n, int act, int precise, int wide, int wanted) {
  Carver c(base);
  Room r = {};
  r.way = ways(rows, k, n, act, precise, wide, wanted);
  const bool z = (wanted == 0 || act != kIdentity) && !r.way.z;
  r.piece = wanted == 0 && r.way.z ? rows : piece_rows(rows, k, n, precise, z);
  if (z) r.z = c.take<float>(r.piece * n);
  if (wanted != 0 && (r.way.z || ((wanted & 3) != 0 && (precise || wide || act != kIdentity)))) r.dz = c.take<__nv_bfloat16>(r.piece * n * (precise ? 3 : 1));
  if (precise && (z || (wanted & 2))) r.x3 = c.take<__nv_bfloat16>(r.piece * k * 3);
  if (precise && (z || (wanted & 1))) r.w3 = c.take<__nv_bfloat16>(3ll * n * k);
  if (wanted & 2) {
    r.per_plane = blocks_per_plane(r.piece, k, n);
    r.splits = r.way.dw ? linear_weights_splits(r.piece, n, k) : weight_splits(r.piece, r.per_plane);
    r.planes = c.take<float>(static_cast<size_t>(r.splits) * n * k);
  }
  if (wanted & 4) {
    const int pairs = r.way.z ? linear_pair_partials(r.piece, n, k) : 0;
    r.partial = c.take<float>(static_cast<size_t>(pairs > kMostRowBlocks ? pairs : kMostRowBlocks) * n);
  }
  r.bytes = c.off;
  return r;
}

MatOperand operand(const void* p, long long ld, int by_k, long long plane) { return {p, ld, by_k, plane}; }

int check(const char* name, long long rows, int k, int n, int act, int dtype) {
  KFB_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && widths_ok(k, n), "%s: rows %lld, %d -> %d channels (multiples of 8)", name, rows, k, n);
  KFB_CHECK_ARG(act >= kIdentity && act <= kRelu, "%s: activation %d", name, act);
  KFB_CHECK_ARG(dtype == KFB_BF16 || dtype == KFB_FP32_PRECISE, "%s: bad dtype %d", name, dtype);
  return KFB_OK;
}
bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API size_t kfb_fused_linear_workspace_bytes(long long rows, int k, int n, int activation, int dtype, int out_dtype, int wanted) {
  if (rows <= 0 || rows >= (1ll << 31) || !widths_ok(k, n)) return 0;
  const int precise = dtype == KFB_FP32_PRECISE;
  return carve(nullptr, rows, k, n, activation, precise, !precise && out_dtype != KFB_BF16, wanted).bytes;
}

KFB_API int kfb_fused_linear_fwd(const void* x, const void* w, const float* bias, const void* residual, void* out, void* workspace,
                                 size_t workspace_bytes, long long rows, int k, int n, int activation, int dtype, int out_dtype, void* stream) {
  KFB_TRY(check("fused_linear", rows, k, n, activation, dtype));
  KFB_CHECK_ARG(out_dtype == KFB_FP32 || (out_dtype == KFB_BF16 && dtype == KFB_BF16), "fused_linear: result of dtype %d", out_dtype);
  if (rows == 0) return KFB_OK;
  const int precise = dtype == KFB_FP32_PRECISE;
  KFB_CHECK_ARG(x != nullptr && w != nullptr && out != nullptr, "fused_linear: null tensor");
  KFB_CHECK_ARG(!off16(x) && !off16(w) && !off16(out) && !off16(residual), "fused_linear: tensors start on 16-byte boundaries");
  const Room m = carve(workspace, rows, k, n, activation, precise, !precise && out_dtype != KFB_BF16, 0);
  cudaStream_t s = as_stream(stream);
  if (m.way.z) {
    const LinearPair p = {kForwardTail, x, w, 0, bias, activation, residual, out, nullptr, rows, n, k};
    return launch_linear_pair(s, p, "fused_linear");
  }
  KFB_CHECK_ARG(workspace != nullptr && workspace_bytes >= m.bytes, "fused_linear: workspace %zu < %zu bytes", workspace_bytes, m.bytes);
  KFB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "fused_linear: workspace must be 256-byte aligned");
  const long long piece = m.piece;
  const size_t out_size = out_dtype == KFB_FP32 ? 4 : 2;
  if (precise) KFB_TRY(launch_split_planes(s, static_cast<const float*>(w), m.w3, static_cast<long long>(n) * k, static_cast<long long>(n) * k));
  for (long long r0 = 0; r0 < rows; r0 += piece) {
    const long long count = rows - r0 < piece ? rows - r0 : piece;
    const uint8_t* xp = static_cast<const uint8_t*>(x) + r0 * k * (precise ? 4 : 2);
    if (precise) KFB_TRY(launch_split_planes(s, reinterpret_cast<const float*>(xp), m.x3, count * k, count * k));
    MatmulArgs a = {};
    a.a = operand(precise ? static_cast<const void*>(m.x3) : xp, k, 0, count * k);
    a.b = operand(precise ? static_cast<const void*>(m.w3) : w, k, 0, static_cast<long long>(n) * k);
    a.m = static_cast<int>(count);
    a.n = n;
    a.k = k;
    a.d = m.z;
    a.ld_d = n;
    a.out_fp32 = 1;
    a.splits = 1;
    a.precise = precise;
    KFB_TRY(launch_matmul(s, a, "fused_linear"));
    TailParams t = {};
    t.z = m.z;
    t.bias = bias;
    t.out_fp32 = t.resid_fp32 = out_dtype == KFB_FP32;
    t.resid = residual != nullptr ? static_cast<const uint8_t*>(residual) + r0 * n * out_size : nullptr;
    t.out = static_cast<uint8_t*>(out) + r0 * n * out_size;
    t.rows = count;
    t.n = n;
    int blocks;
    KFB_TRY(launch_tail<false>(s, t, activation, &blocks));
  }
  return KFB_OK;
}

KFB_API int kfb_fused_linear_bwd(const void* dy, const void* x, const void* w, const float* bias, void* dx, void* dw, float* dbias, void* workspace,
                                 size_t workspace_bytes, long long rows, int k, int n, int activation, int dtype, int dy_dtype, int dw_dtype,
                                 void* stream) {
  KFB_TRY(check("fused_linear_bwd", rows, k, n, activation, dtype));
  const int precise = dtype == KFB_FP32_PRECISE;
  KFB_CHECK_ARG((dy_dtype == KFB_FP32 || (dy_dtype == KFB_BF16 && !precise)) && (dw_dtype == KFB_FP32 || (dw_dtype == KFB_BF16 && !precise)),
                "fused_linear_bwd: dtypes %d and %d", dy_dtype, dw_dtype);
  cudaStream_t s = as_stream(stream);
  if (rows == 0) {
    if (dw != nullptr) KFB_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(n) * k * (dw_dtype == KFB_FP32 ? 4 : 2), s));
    if (dbias != nullptr) KFB_CUDA(cudaMemsetAsync(dbias, 0, static_cast<size_t>(n) * 4, s));
    return KFB_OK;
  }
  const int wanted = (dx != nullptr) + 2 * (dw != nullptr) + 4 * (dbias != nullptr);
  if (wanted == 0) return KFB_OK;
  const bool f = activation != kIdentity, need_z = f;
  KFB_CHECK_ARG(dy != nullptr && (!(dw != nullptr || f) || x != nullptr) && (!(dx != nullptr || f) || w != nullptr), "fused_linear_bwd: null tensor");
  KFB_CHECK_ARG(!off16(dy) && !off16(x) && !off16(w) && !off16(dx) && !off16(dw), "fused_linear_bwd: tensors start on 16-byte boundaries");
  const Room m = carve(workspace, rows, k, n, activation, precise, !precise && dy_dtype != KFB_BF16, wanted);
  KFB_CHECK_ARG(workspace != nullptr || m.bytes == 0, "fused_linear_bwd: null workspace");
  KFB_CHECK_ARG(workspace_bytes >= m.bytes, "fused_linear_bwd: workspace %zu < %zu bytes", workspace_bytes, m.bytes);
  KFB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "fused_linear_bwd: workspace must be 256-byte aligned");
  const long long piece = m.piece, nk = static_cast<long long>(n) * k;
  const size_t dy_size = dy_dtype == KFB_FP32 ? 4 : 2, x_size = precise ? 4 : 2;
  if (m.w3 != nullptr) KFB_TRY(launch_split_planes(s, static_cast<const float*>(w), m.w3, nk, nk));
  for (long long r0 = 0; r0 < rows; r0 += piece) {
    const long long count = rows - r0 < piece ? rows - r0 : piece;
    const uint8_t *xp = static_cast<const uint8_t*>(x) + (x != nullptr ? r0 * k * x_size : 0), *dyp = static_cast<const uint8_t*>(dy) + r0 * n * dy_size;
    if (m.x3 != nullptr) KFB_TRY(launch_split_planes(s, reinterpret_cast<const float*>(xp), m.x3, count * k, count * k));
    const MatOperand xo = operand(precise ? static_cast<const void*>(m.x3) : xp, k, 0, count * k), wo = operand(precise ? static_cast<const void*>(m.w3) : w, k, 0, nk);
    MatmulArgs a = {};
    a.splits = 1;
    a.precise = precise;
    int blocks = 0;
    if (m.way.z) {
      blocks = linear_pair_partials(count, n, k);
      const LinearPair q = {kBackwardTail, xp, w, 0, bias, activation, dyp, m.dz, m.partial, count, n, k};
      KFB_TRY(launch_linear_pair(s, q, "fused_linear_dz"));
    } else if (need_z) {
      a.a = xo;
      a.b = wo;
      a.m = static_cast<int>(count);
      a.n = n;
      a.k = k;
      a.d = m.z;
      a.ld_d = n;
      a.out_fp32 = 1;
      KFB_TRY(launch_matmul(s, a, "fused_linear_z"));
    }
    if (!m.way.z && (m.dz != nullptr || dbias != nullptr)) {
      TailParams t = {};
      t.z = need_z ? m.z : nullptr;
      t.bias = bias;
      t.dy = dyp;
      t.dy_fp32 = dy_dtype == KFB_FP32;
      t.dz = m.dz;
      t.plane = count * n;
      t.parts = precise ? 3 : 1;
      t.partial = m.partial;
      t.rows = count;
      t.n = n;
      KFB_TRY(launch_tail<true>(s, t, activation, &blocks));
    }
    if (dbias != nullptr) {
      LaunchScope scope(s, "linear_bias_sum");
      KFB_TRY(launch_kernel(s, column_sum_kernel, cdiv(n, 32), 1024, 0, const_cast<const float*>(m.partial), dbias, blocks, n, r0 > 0 ? 1 : 0));
    }
    MatOperand dz = operand(m.dz != nullptr ? static_cast<const void*>(m.dz) : dyp, n, 0, count * n);
    if (dx != nullptr && m.way.dx) {
      const LinearPair q = {kPlainTail, dz.ptr, w, 1, nullptr, kIdentity, nullptr, static_cast<uint8_t*>(dx) + r0 * k * x_size, nullptr, count, k, n};
      KFB_TRY(launch_linear_pair(s, q, "fused_linear_dx"));
    } else if (dx != nullptr) {
      a.a = dz;
      a.b = wo;
      a.b.by_k = 1;
      a.m = static_cast<int>(count);
      a.n = k;
      a.k = n;
      a.d = static_cast<uint8_t*>(dx) + r0 * k * x_size;
      a.ld_d = k;
      a.out_fp32 = precise;
      KFB_TRY(launch_matmul(s, a, "fused_linear_dx"));
    }
    if (dw != nullptr && m.way.dw) {
      KFB_TRY(launch_linear_weights(s, dz.ptr, xp, m.planes, m.splits, r0 > 0 ? 1 : 0, count, n, k));
    } else if (dw != nullptr) {
      a.a = dz;
      a.a.by_k = 1;
      a.b = xo;
      a.b.by_k = 1;
      a.m = n;
      a.n = k;
      a.k = count;
      a.d = m.planes;
      a.ld_d = k;
      a.out_fp32 = 1;
      a.splits = weight_splits(count, m.per_plane);
      a.plane_d = nk;
      a.accumulate = r0 > 0;
      KFB_TRY(launch_matmul(s, a, "fused_linear_dw"));
    }
  }
  if (dw != nullptr) {
    const PlaneSum q = {m.planes, nk, m.splits, dw, dw_dtype == KFB_FP32, nk};
    KFB_TRY(launch_sum_planes(s, &q, 1));
  }
  return KFB_OK;
}

}  // extern "C"
