// A linear layer with its tail, and its gradient (training; inference has kfb_gemm_bf16 and kfb_linear_fp32):
//   z = x W^T + b,  y = f(z) (+ residual);   dz = dy f'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz.
//
// z is computed again where f' needs it: 2 of then 8 operations per row and weight, where keeping it is 2 bytes a row and output.  z stays float32;
// dz is rounded to bf16 once, as an operand (dx and dW are then off by 2.4e-3 of their root mean square where their own rounding is 1.7e-3; two bf16 parts would be twice the
// products), and db is summed before that.
// The tail goes with the products: many bf16 rows by CTA pairs (linear_pair.cu), others and the fp32-accurate mode by tiles of 128 x 64 (matmul.cu; those without a tail 128 x 128), dx and dW then
// in one launch.  Rows are taken in pieces, so that the workspace does not grow with them; dW is summed over pieces of rows in float32 planes and added up at the
// end, in an order that depends on the sizes alone.
// float32 (parts of three operands made by launches of their own, six products for one; x's parts are 6 bytes a value, written and read again): 18 432 rows, 384 -> 1 536, forward 270 us (484 TFLOP/s in
// bf16 products; the library's float32 product alone 385), dx and dW with db 292; 384 -> 768 with silu 156 (193) and 301; 147 456 rows of 128 -> 128 154 (115) and 214; 4 096 rows, 384 -> 768,
// sigmoid 43 (62) and 86; 331 rows of 384, silu 15 (11) and 29.
#include "linear_tail.cuh"
#include "matmul.cuh"
#include "ops_common.cuh"

namespace kfb {
namespace {

// ------------------------------------------------------------------------------------------------ dy where nothing is multiplied with it first
constexpr int kCols = 256, kColWarps = 8;            // of a block: a lane has 8 columns of every eighth row
constexpr int kMostRowBlocks = 592;

struct GradientParams {
  const void* dy;
  __nv_bfloat16* dz;           // null, or dy as an operand of the products: rounded, or in three parts `plane` apart
  long long plane;
  float* partial;              // null, or [row block][n] sums of dy
  long long rows;
  int n, rows_per_block, parts, wide;
};

template <bool WIDE>
__global__ void __launch_bounds__(32 * kColWarps) linear_gradient_kernel(const GradientParams p) {
  __shared__ float s[kColWarps][kCols];
  grid_dependency_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * kCols + lane * 8;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const long long first = static_cast<long long>(blockIdx.y) * p.rows_per_block;
  const long long end = first + p.rows_per_block < p.rows ? first + p.rows_per_block : p.rows;
  if (col < p.n) {                                   // (n is a multiple of 8)
#pragma unroll 4
    for (long long r = first + warp; r < end; r += kColWarps) {
      const long long o = r * p.n + col;
      float v[8];
      if constexpr (WIDE) {
        const float4 *q = reinterpret_cast<const float4*>(static_cast<const float*>(p.dy) + o), a = q[0], b = q[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.dy) + o);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += v[i];
      if (p.dz != nullptr) {
        __nv_bfloat16 q[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) split3(v[i], q[0][i], q[1][i], q[2][i]);
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (k < p.parts) *reinterpret_cast<uint4*>(p.dz + k * p.plane + o) = *reinterpret_cast<const uint4*>(q[k]);
      }
    }
  }
  if (p.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[warp][lane * 8 + i] = sum[i];
  __syncthreads();
  const int c = blockIdx.x * kCols + threadIdx.x;
  if (c < p.n) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kColWarps; ++w) t += s[w][threadIdx.x];
    p.partial[static_cast<long long>(blockIdx.y) * p.n + c] = t;
  }
}

int launch_gradient(cudaStream_t stream, GradientParams p, int* row_blocks) {
  const int cols = cdiv(p.n, kCols), most = kMostRowBlocks / cols < 1 ? 1 : kMostRowBlocks / cols;
  long long per = (p.rows + most - 1) / most;
  if (per < kColWarps) per = kColWarps;
  p.rows_per_block = static_cast<int>(per);
  *row_blocks = static_cast<int>((p.rows + per - 1) / per);
  LaunchScope scope(stream, "linear_gradient");
  return p.wide ? launch_kernel(stream, linear_gradient_kernel<true>, dim3(cols, *row_blocks), 32 * kColWarps, 0, p)
                : launch_kernel(stream, linear_gradient_kernel<false>, dim3(cols, *row_blocks), 32 * kColWarps, 0, p);
}

// ------------------------------------------------------------------------------------------------ three bf16 parts of x and W, in one launch
struct SplitPart {
  const float* x;
  __nv_bfloat16* parts;        // [3][n]
  long long n;                 // a multiple of 8
};
struct SplitParams {
  SplitPart s[2];
  unsigned end;                // blocks of the first
};
__global__ void __launch_bounds__(256) linear_split_kernel(const SplitParams p) {
  grid_dependency_enter();
  const int which = blockIdx.x >= p.end;
  const SplitPart& q = p.s[which];
  const long long i = (static_cast<long long>(blockIdx.x - (which ? p.end : 0)) * 256 + threadIdx.x) * 4;
  if (i >= q.n) return;
  const float4 v = *reinterpret_cast<const float4*>(q.x + i);
  const float f[4] = {v.x, v.y, v.z, v.w};
  __nv_bfloat16 t[3][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) split3(f[k], t[0][k], t[1][k], t[2][k]);
#pragma unroll
  for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(q.parts + k * q.n + i) = *reinterpret_cast<const uint2*>(t[k]);
}
int launch_split(cudaStream_t stream, const SplitPart& a, const SplitPart& b) {
  SplitParams p = {{a, b}, 0};
  auto blocks = [](const SplitPart& q) { return q.parts == nullptr ? 0u : static_cast<unsigned>((q.n / 4 + 255) / 256); };
  p.end = blocks(a);
  if (p.end + blocks(b) == 0) return KFB_OK;
  LaunchScope scope(stream, "linear_split");
  return launch_kernel(stream, linear_split_kernel, p.end + blocks(b), 256, 0, p);
}

// ------------------------------------------------------------------------------------------------ sums of planes: dW and db, in one launch
struct Sum {
  const float* planes;         // [count][n]
  int count;
  long long n;                 // a multiple of 8
  void* out;
  int out_fp32, add;
  int parts;                   // launch_sums
};
struct SumParams {
  Sum s[2];
  unsigned end;                // blocks of the first
};
// A block of 256 threads adds up four elements a thread, or `parts` threads add the planes of four elements side by side: where elements are few and planes many
// (the bias's gradient of 63 001 rows of 128 channels 8 us, 47 by one thread each).
constexpr int kSumThreads = 256;
__host__ __device__ constexpr int sum_elements(int parts) { return kSumThreads / parts * 4; }
__global__ void __launch_bounds__(kSumThreads) linear_sum_kernel(const SumParams p) {
  __shared__ float4 s[kSumThreads];
  grid_dependency_enter();
  const int which = blockIdx.x >= p.end;
  const Sum& q = p.s[which];
  const int wide = kSumThreads / q.parts, part = threadIdx.x / wide, lane = threadIdx.x % wide;
  const long long at = static_cast<long long>(blockIdx.x - (which ? p.end : 0)) * sum_elements(q.parts) + lane * 4;
  float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
  if (at < q.n) {
    // (eight planes on their way at a time, the last ones too)
    constexpr int kAhead = 8;
    for (int k = part; k < q.count; k += kAhead * q.parts) {
      float4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int plane = k + j * q.parts;
        v[j] = plane < q.count ? *reinterpret_cast<const float4*>(q.planes + plane * q.n + at) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) t.x += v[j].x, t.y += v[j].y, t.z += v[j].z, t.w += v[j].w;
    }
  }
  if (q.parts > 1) {
    s[threadIdx.x] = t;
    __syncthreads();
    if (part > 0) return;
    for (int k = 1; k < q.parts; ++k) {
      const float4 v = s[k * wide + lane];
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
  }
  if (at >= q.n) return;
  if (q.out_fp32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(q.out) + at);
    if (q.add) {
      const float4 v = *d;
      t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
    *d = t;
  } else {
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(q.out) + at) = make_uint2(pack_bf16x2(t.x, t.y), pack_bf16x2(t.z, t.w));
  }
}
int launch_sums(cudaStream_t stream, const Sum& a, const Sum& b) {
  SumParams p = {{a, b}, 0};
  // as many side by side as give every SM a block, and each more than eight planes to add (dW of 18 432 rows, 384 -> 1 536: 32.1 -> 30.5 us against half as many planes a
  // thread; of 147 456 rows, 512 -> 256: 54.9 -> 52.4 against four blocks an SM)
  for (Sum& q : p.s) {
    q.parts = 1;
    while (q.parts < 64 && q.n * q.parts < kSumThreads * 4 * sm_count() && q.count > 8 * q.parts) q.parts *= 2;
  }
  auto blocks = [](const Sum& q) { return q.out == nullptr ? 0u : static_cast<unsigned>((q.n + sum_elements(q.parts) - 1) / sum_elements(q.parts)); };
  p.end = blocks(p.s[0]);
  const unsigned all = p.end + blocks(p.s[1]);
  if (all == 0) return KFB_OK;
  LaunchScope scope(stream, "linear_sum");
  return launch_kernel(stream, linear_sum_kernel, all, kSumThreads, 0, p);
}

// ------------------------------------------------------------------------------------------------ sizes
bool widths_ok(int k, int n) { return k > 0 && k % 8 == 0 && n > 0 && n % 8 == 0 && k <= 65536 && n <= 65536; }

// Rows of a piece: as many as keep what a row needs in the workspace below half a gigabyte, and 2^30 at most, so that its rows and tiles are counted in 32 bits.
long long piece_rows(long long rows, long long per_row) {
  const long long most = per_row == 0 ? 1ll << 30 : ((1ll << 29) / per_row + 127) / 128 * 128;
  return rows < most ? rows : most;
}

// Blocks of 64 rows that a plane of dW takes from a piece: two tiles an SM, but eight blocks at least: below that a plane costs more than it saves
// (1 024 rows, 384 -> 1 536: 10 us, 15 with two blocks; 8 192 rows of 128 -> 128, where planes are small: 8.5 and 7.9).
int blocks_per_plane(long long piece, int k, int n) {
  const long long tiles = static_cast<long long>(cdiv(n, 128)) * cdiv(k, 128), blocks = (piece + 63) / 64, want = 2 * sm_count() / tiles;
  const long long per = want < 1 ? blocks : (blocks + want - 1) / want;
  return static_cast<int>(per > 8 ? per : blocks < 8 ? blocks : 8);
}
// (a shorter last piece has no more planes than a full one)
int weight_splits(long long rows, int per) { return static_cast<int>(((rows + 63) / 64 + per - 1) / per); }

// How a call goes, and its workspace.  wanted: 0 forward, else a sum of 1 dx, 2 dW, 4 db; wide: the result or its gradient is float32 beside bf16.
struct Plan {
  bool z, again;               // products with a tail: by pairs; at all
  bool dx, dw, ones, whole;    // dx by pairs, dW by pairs, db by dW's kernel, dW in one piece
  long long piece;
  int per_plane, splits;
  __nv_bfloat16 *dz, *x3, *w3;
  float *planes, *partial;
  size_t bytes;
};
Plan plan_of(void* base, long long rows, int k, int n, int act, int precise, int wide, int wanted) {
  Carver c(base);
  Plan p = {};
  p.again = wanted == 0 || act != kIdentity;
  p.z = p.again && !precise && !wide && linear_pair_ok(rows, n, k);
  p.dx = (wanted & 1) && !precise && linear_pair_ok(rows, k, n);
  const bool dz = wanted != 0 && (p.again || ((wanted & 3) != 0 && (precise || wide)));
  const bool x3 = precise && (p.again || (wanted & 2)), w3 = precise && (p.again || (wanted & 1));
  p.piece = piece_rows(rows, (dz ? (precise ? 6ll : 2ll) * n : 0) + (x3 ? 6ll * k : 0));
  const bool ones = (wanted & 4) && !p.again && !wide && p.piece == rows;      // (dW's kernel sums up dy over one piece)
  p.dw = (wanted & 2) && !precise && linear_weights_ok(rows, n, k, ones);
  p.ones = p.dw && ones;
  if (dz) p.dz = c.take<__nv_bfloat16>(p.piece * n * (precise ? 3 : 1));
  if (x3) p.x3 = c.take<__nv_bfloat16>(p.piece * k * 3);
  if (w3) p.w3 = c.take<__nv_bfloat16>(3ll * n * k);
  if (wanted & 2) {
    p.per_plane = blocks_per_plane(p.piece, k, n);
    p.splits = p.dw ? linear_weights_splits(p.piece, n, k) : weight_splits(p.piece, p.per_plane);
    p.whole = !p.dw && p.splits == 1 && p.piece == rows;
    if (!p.whole) p.planes = c.take<float>(static_cast<size_t>(p.splits) * n * k);
  }
  if (wanted & 4) {
    const long long lines = p.ones ? linear_weights_bias_planes(p.splits, k) : p.z ? linear_pair_partials(p.piece, n) : p.again ? 4 * ((p.piece + 127) / 128) : kMostRowBlocks;
    p.partial = c.take<float>(static_cast<size_t>(lines) * n);
  }
  p.bytes = c.off;
  return p;
}

MatOperand operand(const void* p, long long ld, int by_k, long long plane) { return {p, ld, by_k, plane}; }

int check(const char* name, long long rows, int k, int n, int act, int dtype) {
  KFB_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && widths_ok(k, n), "%s: rows %lld, %d -> %d channels (multiples of 8)", name, rows, k, n);
  KFB_CHECK_ARG(act >= kIdentity && act <= kRelu, "%s: activation %d", name, act);
  KFB_CHECK_ARG(dtype == KFB_BF16 || dtype == KFB_FP32_PRECISE, "%s: bad dtype %d", name, dtype);
  return KFB_OK;
}
int check_room(const char* name, const Plan& m, const void* workspace, size_t bytes) {
  KFB_CHECK_ARG(m.bytes == 0 || (workspace != nullptr && bytes >= m.bytes), "%s: workspace %zu < %zu bytes", name, bytes, m.bytes);
  KFB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "%s: workspace must be 256-byte aligned", name);
  return KFB_OK;
}
bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// z = x W^T with a tail, by tiles of 128 x 64.
int launch_tail(cudaStream_t s, const MatOperand& x, const MatOperand& w, const MatmulTail& tail, void* d, int out_fp32, long long plane, long long rows, int k, int n,
                int precise, const char* tag) {
  MatmulArgs a = {};
  a.a = x;
  a.b = w;
  a.m = static_cast<int>(rows);
  a.n = n;
  a.k = k;
  a.d = d;
  a.ld_d = n;
  a.out_fp32 = out_fp32;
  a.splits = 1;
  a.plane_d = plane;
  a.precise = precise;
  a.turns = kMostTurns;
  a.tail = &tail;
  return launch_matmul(s, a, tag);
}

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API size_t kfb_fused_linear_workspace_bytes(long long rows, int k, int n, int activation, int dtype, int out_dtype, int wanted) {
  if (rows <= 0 || rows >= (1ll << 31) || !widths_ok(k, n)) return 0;
  const int precise = dtype == KFB_FP32_PRECISE;
  return plan_of(nullptr, rows, k, n, activation, precise, !precise && out_dtype != KFB_BF16, wanted).bytes;
}

KFB_API int kfb_fused_linear_fwd(const void* x, const void* w, const float* bias, const void* residual, void* out, void* workspace,
                                 size_t workspace_bytes, long long rows, int k, int n, int activation, int dtype, int out_dtype, void* stream) {
  KFB_TRY(check("fused_linear", rows, k, n, activation, dtype));
  KFB_CHECK_ARG(out_dtype == KFB_FP32 || (out_dtype == KFB_BF16 && dtype == KFB_BF16), "fused_linear: result of dtype %d", out_dtype);
  if (rows == 0) return KFB_OK;
  const int precise = dtype == KFB_FP32_PRECISE, wide = out_dtype == KFB_FP32;
  KFB_CHECK_ARG(x != nullptr && w != nullptr && out != nullptr, "fused_linear: null tensor");
  KFB_CHECK_ARG(!off16(x) && !off16(w) && !off16(bias) && !off16(out) && !off16(residual), "fused_linear: tensors start on 16-byte boundaries");
  const Plan m = plan_of(workspace, rows, k, n, activation, precise, !precise && wide, 0);
  KFB_TRY(check_room("fused_linear", m, workspace, workspace_bytes));
  cudaStream_t s = as_stream(stream);
  if (m.z) {
    const LinearPair p = {kForwardTail, x, w, 0, bias, activation, residual, out, nullptr, rows, n, k};
    return launch_linear_pair(s, p, "fused_linear");
  }
  const long long nk = static_cast<long long>(n) * k;
  const size_t out_size = wide ? 4 : 2, x_size = precise ? 4 : 2;
  for (long long r0 = 0; r0 < rows; r0 += m.piece) {
    const long long count = rows - r0 < m.piece ? rows - r0 : m.piece;
    const uint8_t* xp = static_cast<const uint8_t*>(x) + r0 * k * x_size;
    if (precise)
      KFB_TRY(launch_split(s, {reinterpret_cast<const float*>(xp), m.x3, count * k}, {static_cast<const float*>(w), r0 == 0 ? m.w3 : nullptr, nk}));
    const MatmulTail tail = {0, activation, bias, residual != nullptr ? static_cast<const uint8_t*>(residual) + r0 * n * out_size : nullptr, wide, 1, nullptr};
    KFB_TRY(launch_tail(s, operand(precise ? static_cast<const void*>(m.x3) : xp, k, 0, count * k), operand(precise ? static_cast<const void*>(m.w3) : w, k, 0, nk), tail,
                        static_cast<uint8_t*>(out) + r0 * n * out_size, wide, 0, count, k, n, precise, "fused_linear"));
  }
  return KFB_OK;
}

KFB_API int kfb_fused_linear_bwd(const void* dy, const void* x, const void* w, const float* bias, void* dx, void* dw, float* dbias, void* workspace,
                                 size_t workspace_bytes, long long rows, int k, int n, int activation, int dtype, int dy_dtype, int dw_dtype,
                                 void* stream) {
  KFB_TRY(check("fused_linear_bwd", rows, k, n, activation, dtype));
  const int precise = dtype == KFB_FP32_PRECISE, wide = dy_dtype == KFB_FP32;
  KFB_CHECK_ARG((wide || (dy_dtype == KFB_BF16 && !precise)) && (dw_dtype == KFB_FP32 || (dw_dtype == KFB_BF16 && !precise)),
                "fused_linear_bwd: dtypes %d and %d", dy_dtype, dw_dtype);
  cudaStream_t s = as_stream(stream);
  if (rows == 0) {
    if (dw != nullptr) KFB_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(n) * k * (dw_dtype == KFB_FP32 ? 4 : 2), s));
    if (dbias != nullptr) KFB_CUDA(cudaMemsetAsync(dbias, 0, static_cast<size_t>(n) * 4, s));
    return KFB_OK;
  }
  const int wanted = (dx != nullptr) + 2 * (dw != nullptr) + 4 * (dbias != nullptr);
  if (wanted == 0) return KFB_OK;
  const bool f = activation != kIdentity;
  KFB_CHECK_ARG(dy != nullptr && (!(dw != nullptr || f) || x != nullptr) && (!(dx != nullptr || f) || w != nullptr), "fused_linear_bwd: null tensor");
  KFB_CHECK_ARG(!off16(dy) && !off16(x) && !off16(w) && !off16(bias) && !off16(dx) && !off16(dw) && !off16(dbias),
                "fused_linear_bwd: tensors start on 16-byte boundaries");
  const Plan m = plan_of(workspace, rows, k, n, activation, precise, !precise && wide, wanted);
  KFB_TRY(check_room("fused_linear_bwd", m, workspace, workspace_bytes));
  const long long nk = static_cast<long long>(n) * k;
  const size_t dy_size = wide ? 4 : 2, x_size = precise ? 4 : 2;
  for (long long r0 = 0; r0 < rows; r0 += m.piece) {
    const long long count = rows - r0 < m.piece ? rows - r0 : m.piece;
    const bool last = r0 + count == rows;
    const uint8_t *xp = x != nullptr ? static_cast<const uint8_t*>(x) + r0 * k * x_size : nullptr, *dyp = static_cast<const uint8_t*>(dy) + r0 * n * dy_size;
    KFB_TRY(launch_split(s, {reinterpret_cast<const float*>(xp), m.x3, count * k}, {static_cast<const float*>(w), r0 == 0 ? m.w3 : nullptr, nk}));
    const MatOperand xo = operand(precise ? static_cast<const void*>(m.x3) : xp, k, 0, count * k), wo = operand(precise ? static_cast<const void*>(m.w3) : w, k, 0, nk);
    float* partial = m.ones ? nullptr : m.partial;
    int lines = 0;                                   // of partial sums
    if (m.z) {
      const LinearPair q = {kBackwardTail, xp, w, 0, bias, activation, dyp, m.dz, partial, count, n, k};
      lines = linear_pair_partials(count, n);
      KFB_TRY(launch_linear_pair(s, q, "fused_linear_dz"));
    } else if (m.again) {
      const MatmulTail tail = {1, activation, bias, dyp, wide, precise ? 3 : 1, partial};
      lines = 4 * cdiv(static_cast<int>(count), 128);
      KFB_TRY(launch_tail(s, xo, wo, tail, m.dz, 0, count * n, count, k, n, precise, "fused_linear_dz"));
    } else if (m.dz != nullptr || partial != nullptr) {
      GradientParams g = {};
      g.dy = dyp;
      g.dz = m.dz;
      g.plane = count * n;
      g.partial = partial;
      g.rows = count;
      g.n = n;
      g.parts = precise ? 3 : 1;
      g.wide = wide;
      KFB_TRY(launch_gradient(s, g, &lines));
    }
    // dx and dW: one launch where neither goes by pairs
    const MatOperand dz = operand(m.dz != nullptr ? static_cast<const void*>(m.dz) : dyp, n, 0, count * n);
    MatmulArgs list[2] = {};
    int products = 0;
    if (dx != nullptr && m.dx) {
      const LinearPair q = {kPlainTail, dz.ptr, w, 1, nullptr, kIdentity, nullptr, static_cast<uint8_t*>(dx) + r0 * k * x_size, nullptr, count, k, n};
      KFB_TRY(launch_linear_pair(s, q, "fused_linear_dx"));
    } else if (dx != nullptr) {
      MatmulArgs& a = list[products++];
      a.a = dz;
      a.b = wo;
      a.b.by_k = 1;
      a.m = static_cast<int>(count);
      a.n = k;
      a.k = n;
      a.d = static_cast<uint8_t*>(dx) + r0 * k * x_size;
      a.ld_d = k;
      a.out_fp32 = precise;
      a.splits = 1;
      a.precise = precise;
      a.turns = kMostTurns;
    }
    if (dw != nullptr && m.dw) {
      KFB_TRY(launch_linear_weights(s, dz.ptr, xp, m.planes, m.ones ? m.partial : nullptr, m.splits, r0 > 0 ? 1 : 0, count, n, k));
      if (m.ones) lines = linear_weights_bias_planes(m.splits, k);
    } else if (dw != nullptr) {
      MatmulArgs& a = list[products++];
      a.a = dz;
      a.a.by_k = 1;
      a.b = xo;
      a.b.by_k = 1;
      a.m = n;
      a.n = k;
      a.k = count;
      a.d = m.whole ? dw : m.planes;
      a.ld_d = k;
      a.out_fp32 = !m.whole || dw_dtype == KFB_FP32;
      a.splits = weight_splits(count, m.per_plane);
      a.plane_d = nk;
      a.accumulate = r0 > 0;
      a.precise = precise;
      a.turns = kMostTurns;
    }
    if (products > 0) KFB_TRY(launch_matmuls(s, list, products, "fused_linear_grads"));
    Sum of_w = {m.planes, m.splits, nk, last && !m.whole ? dw : nullptr, dw_dtype == KFB_FP32, 0, 1};
    // (dW's planes hold the pieces before, db's are a piece's own)
    Sum of_b = {m.partial, lines, n, dbias, 1, r0 > 0, 1};
    KFB_TRY(launch_sums(s, of_w, of_b));
  }
  return KFB_OK;
}

}  // extern "C"
