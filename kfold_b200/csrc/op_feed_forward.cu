// Gated feed-forward and its gradient (training; the inference path has it inside kfb_transition_fwd):
//   [a, b] = x [Wa; Wb]^T,  h = silu(a) b,  y = h Wo^T
//   dh = dy Wo,  da = dh b silu'(a),  db = dh silu(a),  dx = [da, db] [Wa; Wb],  d[Wa; Wb] = [da, db]^T x,  dWo = dy^T h
// with s = sigmoid(a), silu(a) = a s, silu'(a) = s + silu(a) (1 - s).
//
// a and b are not kept from the forward pass: computing them again is 4 of the backward pass's 16 operations per row, channel and hidden channel,
// keeping them 8 bytes per row and hidden channel.  a, b and dh stay float32; h, da and db are rounded to bf16 once, as operands.
// Rows are taken in pieces, so that the workspace does not grow with them; the weights' gradients are summed over pieces of rows in float32
// planes and added up at the end, in an order that depends on the sizes alone.
#include "feed_forward_hidden.cuh"
#include "gemm.cuh"   // sigmoidf_exact, split3
#include "matmul.cuh"
#include "ops_common.cuh"
#include "transition_pair.cuh"

namespace kfb {
namespace {

// The widths that the sizes below are computed for without leaving their range.
bool widths_ok(int c, int hidden) { return c > 0 && c % 8 == 0 && hidden > 0 && hidden % 8 == 0 && c <= 65536 && hidden <= 65536; }

// Rows of a piece: as many as keep what a row needs between its products below a gigabyte.  (Smaller ones, whose hidden channels would stay in L2, are no
// faster: writes into L2 are no faster than writes through it, and every piece starts and ends its launches.)
long long piece_rows(long long rows, int c, int hidden, int precise, int backward, bool one) {
  const long long per_row = precise ? 12ll * c + (backward ? 30ll : 14ll) * hidden : one ? (backward ? 6ll : 2ll) * hidden : (backward ? 18ll : 10ll) * hidden;
  const long long most = ((1ll << 30) / per_row + 255) / 256 * 256;
  return rows < most ? rows : most;
}

// h and, with dh, [da, db] from u = [a, b] (rows, 2 hidden) and dh (rows, hidden); four hidden channels a thread.  PARTS == 3: the results as three
// bf16 parts each, planes rows * hidden and rows * 2 hidden apart.
template <int PARTS>
__device__ __forceinline__ void store_parts(__nv_bfloat16* d, long long plane, const float (&v)[4]) {
  if constexpr (PARTS == 1) {
    *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  } else {
    __nv_bfloat16 q[3][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) split3(v[k], q[0][k], q[1][k], q[2][k]);
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(d + k * plane) = *reinterpret_cast<const uint2*>(q[k]);
  }
}

template <int PARTS>
__global__ void __launch_bounds__(256) ffn_hidden_kernel(const float* u, const float* dh, __nv_bfloat16* h, __nv_bfloat16* dab, long long rows,
                                                         int hidden) {
  grid_dependency_enter();
  const long long per_row = hidden / 4, n = rows * per_row;
  for (long long t = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; t < n; t += static_cast<long long>(gridDim.x) * 256) {
    const long long row = t / per_row;
    const int j = static_cast<int>(t - row * per_row) * 4;
    const float4 a4 = *reinterpret_cast<const float4*>(u + row * 2 * hidden + j), b4 = *reinterpret_cast<const float4*>(u + row * 2 * hidden + hidden + j);
    const float4 g4 = dh != nullptr ? *reinterpret_cast<const float4*>(dh + row * hidden + j) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
    float hv[4], da[4], db[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float s = sigmoidf_exact(a[i]), silu = a[i] * s;
      hv[i] = silu * b[i];
      da[i] = g[i] * b[i] * fmaf(silu, 1.0f - s, s);
      db[i] = g[i] * silu;
    }
    store_parts<PARTS>(h + row * hidden + j, rows * hidden, hv);
    if (dh != nullptr) {
      store_parts<PARTS>(dab + row * 2 * hidden + j, rows * 2 * hidden, da);
      store_parts<PARTS>(dab + row * 2 * hidden + hidden + j, rows * 2 * hidden, db);
    }
  }
}

struct FfnWs {
  __nv_bfloat16 *x3, *dy3, *wi3, *wo3;      // fp32-accurate mode: the operands' parts
  float *u, *dh;                            // where no kernel keeps them in tensor memory
  __nv_bfloat16 *h, *dab, *wi_t;
  float *pl_in, *pl_out, *pl_dx;
};
// Whether h, da and db come from the one kernel (feed_forward_hidden.cu).
bool one_kernel(int c, int hidden, int precise) { return !precise && ffn_hidden_ok(c, hidden); }
// Whether there are rows enough for the kernels of 256-row tiles that have dx with the hidden channels (feed_forward_rows.cu) and the weights' sums
// (feed_forward_weights.cu, feed_forward_sums.cu).  Few do not fill them: the kernel that spreads the hidden channels over the device, and one launch of all
// products, are faster.  Gradient alone, these and the one launch: 128 channels, 512 hidden, 4 000 rows 26 and 21 us, 7 200 29 and 25, 9 500 31 and 32, 20 000 46 and 58;
// 256 channels, 1 024 hidden, 7 200 rows 63 and 45, 9 500 66 and 73, 20 000 117 and 154.  Fewer hidden channels shorten the one launch more: 128 and 256,
// 16 000 rows 31 and 26, 30 000 40 and 45; 256 and 512, 12 000 rows 48 and 46, 18 900 54 and 60.
bool many_rows(long long rows, int c, int hidden) { return rows >= 64ll * sm_count() && rows * hidden >= 64ll * sm_count() * 4 * c; }
// Whether both gradients come from x and dy alone, nothing kept in between.
bool nothing_kept(long long rows, int c, int hidden, int precise) {
  return !precise && many_rows(rows, c, hidden) && ffn_weights_ok(c, hidden) && ffn_rows_ok(c, hidden);
}
bool sums_kernel(long long piece, int c, int hidden, int precise) {
  return many_rows(piece, c, hidden) && one_kernel(c, hidden, precise) && ffn_sums_ok(c, hidden);
}

// What a call is asked for: its result, or some of the gradients (the entry point's `wanted`).
constexpr int kForward = 0, kDx = 1, kDwIn = 2, kDwOut = 4, kAll = 7;
// Whether the forward pass is the pair kernel's, which keeps nothing, or two launches.  The rule is the Transition's, whose other form has a LayerNorm's
// launch more.  Pair kernel and two launches, graph replays, us:
//   128 channels, 512 hidden      64 rows 8.6 and 8.7, 1 024 9.4 and 9.4, 8 192 9.9 and 13.1, 63 001 23 and 40
//   128 channels, 1 024 hidden    1 024 rows 13.1 and 11.9 (takes two), 2 048 13.3 and 12.9 (pair), 4 096 13.5 and 14.7, 63 001 40 and 78
//   256 channels, 512 hidden      4 096 rows 14.1 and 12.3 (two), 5 000 14.1 and 12.6 (pair), 7 000 14.2 and 14.0, 9 600 14.7 and 18.3, 63 001 41 and 55
//   256 channels, 1 024 hidden    8 192 rows 22.3 and 19.6 (two), 9 000 22.4 and 19.9 (pair), 9 600 22.9 and 27.5, 19 000 39 and 45, 63 001 73 and 101
//   256 channels, 2 048 hidden    9 000 rows 38 and 31 (two), 9 600 39 and 46 (pair), 19 000 71 and 85 (two), 22 000 72 and 90 (pair)
// So it takes the slower form by up to an eighth for 5 000 to 6 500 and 8 500 to 9 500 rows of 256 channels, and by a fifth for 19 000 to 21 000 of 2 048 hidden.
bool forward_by_pair(long long rows, int c, int hidden, int precise) {
  return !precise && feed_forward_pair_ok(rows, c, hidden) && transition_pair_is_faster(rows, c, hidden);
}
// Whether m rows of a gradient that keeps hidden channels for the weights' sums have dx from the kernel that computes them.
bool dx_with_hidden(long long m, int c, int hidden, bool one) { return one && c == 256 && ffn_rows_ok(c, hidden) && many_rows(m, c, hidden); }

// How the products of a gradient that share a launch are cut along their contractions: dx (`dx_tiles` tiles of dx_k blocks of 64) and the weights' gradients
// (`w_tiles` of w_k).  Pieces fill the device, but each starts and ends, and writes a float32 plane that is read again.  So the cheapest of these counts by
// the time that a launch takes: its blocks, side by side on an SM, two where they fit; waves of them; planes; the launch that adds them up.  The four
// rates are fitted to 2 300 launches (50 ... 20 000 rows of 64 ... 768 channels): on average 2 % longer than the best count of each, 9 % at most.  Each product
// cut as if it had the device to itself was 21 % longer: 3 000 rows of 384 channels 59 us for the whole gradient, 36 by these (uncut), 4 000 of 256
// 46 and 34, 2 000 of 768 90 and 77, 331 of 384 17 and 18.
struct Cuts {
  int dx, w;
};
Cuts best_cuts(int dx_tiles, int dx_k, bool cut_dx, int w_tiles, int w_k, int precise) {
  static constexpr int kDx[] = {1, 2, 4, 8}, kW[] = {1, 2, 3, 4, 8, 16, 32, 64}, kLeast = 4;      // (a piece has four blocks at least)
  const float sms = static_cast<float>(sm_count()), at_once = precise ? 1.f : 2.f;      // (the fp32-accurate mode's blocks fill an SM, and take six products for one)
  const float per_block = precise ? 0.7f : 0.117f, per_wave = 4.7f, per_plane = 0.0205f, per_sum = 1.3f;      // us
  Cuts best = {1, 1};
  float least = 0.f;
  for (int i = 0; i < (cut_dx ? 4 : 1); ++i) {
    if (i > 0 && dx_k < kDx[i] * kLeast) break;
    const int dx_len = cdiv(dx_k, kDx[i]), dx_n = cdiv(dx_k, dx_len);
    for (int j = 0; j < 8; ++j) {
      if (j > 0 && w_k < kW[j] * kLeast) break;
      const int w_len = cdiv(w_k, kW[j]), w_n = cdiv(w_k, w_len);
      const float d = static_cast<float>(dx_tiles) * dx_n, w = static_cast<float>(w_tiles) * w_n, n = d + w;
      const float longest = static_cast<float>(dx_tiles > 0 && dx_len > w_len ? dx_len : w_len);
      const float planes = (dx_n > 1 ? d : 0.f) + (w_n > 1 ? w : 0.f);
      const float share = (d * dx_len + w * w_len) / sms, side = n / sms < 1.f ? 1.f : n / sms < at_once ? n / sms : at_once;
      const float waves = n / (at_once * sms);
      const float t = per_block * (share > longest * side ? share : longest * side) + per_wave * (waves > 1.f ? waves : 1.f) + per_plane * planes +
                      (planes > 0.f ? per_sum : 0.f);
      if ((i == 0 && j == 0) || t < least) {
        least = t;
        best = {dx_n, w_n};
      }
    }
  }
  return best;
}
// `most` pieces of `blocks`, fewer where some would be empty.
int pieces_of(int blocks, int most) { return cdiv(blocks, cdiv(blocks, most < blocks ? most : blocks)); }

// What the gradient of these sizes does, whoever asks for which of its results.
struct Plan {
  long long piece;       // rows
  bool one, sums_by_pair;
  bool dx_here;          // dx by the launch of the weights' gradients (few rows), or by the library's own product for operands along k
  int in, out, dx;       // float32 planes of dw_in and dw_out (1: none, where the rows come in one piece), and of dx
};
Plan plan_of(long long rows, int c, int hidden, int precise) {
  Plan p = {};
  p.one = one_kernel(c, hidden, precise);
  p.piece = piece_rows(rows, c, hidden, precise, 1, p.one);
  p.sums_by_pair = sums_kernel(p.piece, c, hidden, precise);
  const bool single = rows <= p.piece;
  const long long dx_tiles = static_cast<long long>(cdiv(static_cast<int>(p.piece), 128)) * cdiv(c, 128);
  p.dx_here = precise || (single && dx_tiles < 2 * sm_count());
  const int w_tiles = cdiv(c, 128) * (cdiv(2 * hidden, 128) + cdiv(hidden, 128));
  const Cuts cuts = best_cuts(p.dx_here ? static_cast<int>(dx_tiles) : 0, cdiv(2 * hidden, 64), p.dx_here && single, p.sums_by_pair ? 0 : w_tiles,
                              p.sums_by_pair ? 1 : cdiv(static_cast<int>(p.piece), 64), precise);
  p.in = p.out = p.sums_by_pair ? ffn_sums_planes(p.piece, hidden) : cuts.w;
  p.dx = cuts.dx;
  return p;
}

// The workspace of a gradient by `p` that is asked for `wanted`.
size_t carve_gradient(FfnWs& w, void* base, long long rows, int c, int hidden, int precise, const Plan& p, int wanted) {
  Carver cv(base);
  const size_t cc = c, hh = hidden;
  w = {};
  if (nothing_kept(rows, c, hidden, precise)) {
    const size_t planes = ffn_weights_planes(rows, hidden);
    if (wanted & kDwIn) w.pl_in = cv.take<float>(planes * 2 * hh * cc);
    if (wanted & kDwOut) w.pl_out = cv.take<float>(planes * hh * cc);
    return cv.off;
  }
  // Rows whose hidden channels lie in memory between launches: a piece; where dx alone is wanted and has a kernel of its own, those of a last piece
  // that is too short for it, if any.
  const long long last = rows % p.piece;
  auto by_rows = [&](long long m) { return (wanted & kDx) != 0 && dx_with_hidden(m, c, hidden, p.one); };
  auto kept = [&](long long m) { return m > 0 && ((wanted & (kDwIn | kDwOut)) != 0 || !by_rows(m)); };
  const size_t r = static_cast<size_t>(kept(p.piece) ? p.piece : kept(last) ? last : 0), parts = precise ? 3 : 1;
  const bool single = rows <= p.piece;
  if (precise) {
    w.x3 = cv.take<__nv_bfloat16>(3 * r * cc);
    w.wi3 = cv.take<__nv_bfloat16>(3 * 2 * hh * cc);
    w.wo3 = cv.take<__nv_bfloat16>(3 * hh * cc);
    w.dy3 = cv.take<__nv_bfloat16>(3 * r * cc);
  }
  if (!p.one) {
    w.u = cv.take<float>(r * 2 * hh);
    w.dh = cv.take<float>(r * hh);
  }
  w.h = cv.take<__nv_bfloat16>(parts * r * hh);
  w.dab = cv.take<__nv_bfloat16>(parts * r * 2 * hh);
  if ((wanted & kDx) && !p.dx_here && r > 0) w.wi_t = cv.take<__nv_bfloat16>(2 * hh * cc);
  if ((wanted & kDwIn) && (p.sums_by_pair || !single || p.in > 1)) w.pl_in = cv.take<float>(p.in * 2 * hh * cc);
  if ((wanted & kDwOut) && (p.sums_by_pair || !single || p.out > 1)) w.pl_out = cv.take<float>(p.out * hh * cc);
  if ((wanted & kDx) && p.dx > 1) w.pl_dx = cv.take<float>(p.dx * r * cc);
  return cv.off;
}
// ... of the forward pass by the launches that keep h.
size_t carve_forward(FfnWs& w, void* base, long long rows, int c, int hidden, int precise) {
  Carver cv(base);
  const bool one = one_kernel(c, hidden, precise);
  const size_t r = static_cast<size_t>(piece_rows(rows, c, hidden, precise, 0, one)), parts = precise ? 3 : 1, cc = c, hh = hidden;
  w = {};
  if (precise) {
    w.x3 = cv.take<__nv_bfloat16>(3 * r * cc);
    w.wi3 = cv.take<__nv_bfloat16>(3 * 2 * hh * cc);
    w.wo3 = cv.take<__nv_bfloat16>(3 * hh * cc);
  }
  if (!one) w.u = cv.take<float>(r * 2 * hh);
  w.h = cv.take<__nv_bfloat16>(parts * r * hh);
  return cv.off;
}

int launch_hidden(cudaStream_t stream, const FfnWs& w, bool backward, long long rows, int hidden, int precise) {
  const long long want = (rows * (hidden / 4) + 255) / 256, most = static_cast<long long>(sm_count()) * 16;
  LaunchScope scope(stream, "feed_forward_hidden");
  return launch_kernel(stream, precise ? ffn_hidden_kernel<3> : ffn_hidden_kernel<1>, static_cast<unsigned>(want < most ? want : most), 256, 0,
                       const_cast<const float*>(w.u), backward ? const_cast<const float*>(w.dh) : nullptr, w.h, w.dab, rows, hidden);
}

// t[j][i] = w[i][j], 32 x 32 a block
__global__ void __launch_bounds__(256) transpose_kernel(const __nv_bfloat16* w, __nv_bfloat16* t, int rows, int cols) {
  __shared__ __nv_bfloat16 s[32][34];
  grid_dependency_enter();
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32, i = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int k = i; k < 32; k += 8)
    if (r0 + k < rows && c0 + lane < cols) s[k][lane] = w[static_cast<long long>(r0 + k) * cols + c0 + lane];
  __syncthreads();
#pragma unroll
  for (int k = i; k < 32; k += 8)
    if (c0 + k < cols && r0 + lane < rows) t[static_cast<long long>(c0 + k) * rows + r0 + lane] = s[lane][k];
}
int launch_transpose(cudaStream_t stream, const void* w, __nv_bfloat16* t, int rows, int cols) {
  LaunchScope scope(stream, "feed_forward_transpose");
  return launch_kernel(stream, transpose_kernel, dim3(cdiv(cols, 32), cdiv(rows, 32)), 256, 0, static_cast<const __nv_bfloat16*>(w), t, rows, cols);
}

// out = a b^T, a (m, k), b (n, k): the library's own product for operands along k
int product(cudaStream_t stream, const void* a, const void* b, void* out, long long m, int n, int k, const char* tag) {
  GemmParams p = {};
  p.n_extent = static_cast<int>(m);
  p.o_extent = 1;
  p.batch = 1;
  p.n_cols = n;
  p.k_extent = k;
  p.nseg = 1;
  p.seg[0] = row_major_seg(out, n, n, 0, 0, 0);
  GemmOperandA oa = {a, k, 0, 0};
  GemmOperandB ob = {b, k, 0};
  return launch_gemm_bf16(stream, oa, ob, p, 0, tag);
}

int check(const char* name, const void* workspace, size_t workspace_bytes, size_t need, long long rows, int c, int hidden, int dtype,
          uintptr_t tensors) {
  KFB_CHECK_ARG(dtype == KFB_BF16 || dtype == KFB_FP32_PRECISE, "%s: bad dtype %d", name, dtype);
  KFB_CHECK_ARG(rows >= 0 && rows < (1ll << 31), "%s: rows %lld", name, rows);
  KFB_CHECK_ARG(widths_ok(c, hidden), "%s: c=%d, hidden=%d (multiples of 8 up to 65 536)", name, c, hidden);
  KFB_CHECK_ARG((tensors & 15) == 0, "%s: tensors must be 16-byte aligned", name);
  KFB_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need), "%s: workspace %zu < %zu bytes", name, workspace_bytes, need);
  KFB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "%s: workspace must be 256-byte aligned", name);
  return KFB_OK;
}
uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API size_t kfb_feed_forward_call_bytes(long long rows, int c, int hidden, int dtype, int wanted) {
  if (rows < 1 || rows >= (1ll << 31) || !widths_ok(c, hidden) || wanted < kForward || wanted > kAll) return 0;
  const int precise = dtype == KFB_FP32_PRECISE;
  FfnWs w;
  if (wanted == kForward) return forward_by_pair(rows, c, hidden, precise) ? 0 : carve_forward(w, nullptr, rows, c, hidden, precise);
  return carve_gradient(w, nullptr, rows, c, hidden, precise, plan_of(rows, c, hidden, precise), wanted);
}

KFB_API size_t kfb_feed_forward_workspace_bytes(long long rows, int c, int hidden, int dtype, int backward) {
  if (rows < 1 || !widths_ok(c, hidden)) return 0;
  const int precise = dtype == KFB_FP32_PRECISE;
  FfnWs w;
  return backward ? carve_gradient(w, nullptr, rows, c, hidden, precise, plan_of(rows, c, hidden, precise), kAll)
                  : carve_forward(w, nullptr, rows, c, hidden, precise);
}

KFB_API int kfb_feed_forward_fwd(const void* x, const void* w_in, const void* w_out, void* out, void* workspace, size_t workspace_bytes,
                                 long long rows, int c, int hidden, int dtype, void* stream) {
  if (rows == 0) return KFB_OK;
  KFB_CHECK_ARG(x && w_in && w_out && out, "feed_forward: null tensor");
  KFB_TRY(check("feed_forward", workspace, workspace_bytes, kfb_feed_forward_call_bytes(rows, c, hidden, dtype, kForward), rows, c, hidden, dtype,
                bits(x) | bits(w_in) | bits(w_out) | bits(out)));
  cudaStream_t s = as_stream(stream);
  const int precise = dtype == KFB_FP32_PRECISE;
  const size_t size = precise ? 4 : 2;
  if (forward_by_pair(rows, c, hidden, precise)) return launch_feed_forward_pair(s, x, w_in, w_out, out, rows, c, hidden);
  FfnWs w;
  carve_forward(w, workspace, rows, c, hidden, precise);
  const long long wi_n = 2ll * hidden * c, wo_n = static_cast<long long>(hidden) * c;
  if (precise) {
    KFB_TRY(launch_split_planes(s, static_cast<const float*>(w_in), w.wi3, wi_n, wi_n));
    KFB_TRY(launch_split_planes(s, static_cast<const float*>(w_out), w.wo3, wo_n, wo_n));
  }
  const void *wi = precise ? w.wi3 : w_in, *wo = precise ? w.wo3 : w_out;
  const bool one = one_kernel(c, hidden, precise);
  const long long piece = piece_rows(rows, c, hidden, precise, 0, one);
  for (long long r0 = 0; r0 < rows; r0 += piece) {
    const long long r = rows - r0 < piece ? rows - r0 : piece;
    const int m = static_cast<int>(r);
    const void* xr = static_cast<const char*>(x) + r0 * c * size;
    if (one) {
      KFB_TRY(launch_ffn_hidden(s, xr, nullptr, wi, wo, w.h, nullptr, m, c, hidden));
      KFB_TRY(product(s, w.h, wo, static_cast<char*>(out) + r0 * c * size, r, c, hidden, "feed_forward_out"));
      continue;
    }
    if (precise) {
      KFB_TRY(launch_split_planes(s, static_cast<const float*>(xr), w.x3, r * c, r * c));
      xr = w.x3;
    }
    MatmulArgs in = {{xr, c, 0, r * c}, {wi, c, 0, wi_n}, m, 2 * hidden, c, w.u, 2ll * hidden, 1, 1, 0, 0, precise};
    KFB_TRY(launch_matmul(s, in, "feed_forward_in"));
    KFB_TRY(launch_hidden(s, w, false, r, hidden, precise));
    MatmulArgs out_p = {{w.h, hidden, 0, r * hidden}, {wo, hidden, 0, wo_n}, m, c, hidden, static_cast<char*>(out) + r0 * c * size, c, precise, 1, 0, 0,
                        precise};
    KFB_TRY(launch_matmul(s, out_p, "feed_forward_out"));
  }
  return KFB_OK;
}

KFB_API int kfb_feed_forward_bwd(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx, void* dw_in, void* dw_out,
                                 void* workspace, size_t workspace_bytes, long long rows, int c, int hidden, int dtype, int grad_dtype,
                                 void* stream) {
  cudaStream_t s = as_stream(stream);
  const long long wi_n = 2ll * hidden * c, wo_n = static_cast<long long>(hidden) * c;
  const int precise = dtype == KFB_FP32_PRECISE;
  const size_t size = precise ? 4 : 2;
  KFB_CHECK_ARG(grad_dtype == KFB_FP32 || (grad_dtype == KFB_BF16 && !precise), "feed_forward_bwd: bad dtype %d of the weights' gradients", grad_dtype);
  if (rows == 0) {
    const size_t g = grad_dtype == KFB_FP32 ? 4 : 2;
    KFB_CHECK_ARG(widths_ok(c, hidden), "feed_forward_bwd: c=%d, hidden=%d (multiples of 8 up to 65 536)", c, hidden);
    if (dw_in != nullptr) KFB_CUDA(cudaMemsetAsync(dw_in, 0, wi_n * g, s));
    if (dw_out != nullptr) KFB_CUDA(cudaMemsetAsync(dw_out, 0, wo_n * g, s));
    return KFB_OK;
  }
  KFB_CHECK_ARG(dy && x && w_in && w_out, "feed_forward_bwd: null tensor");
  const bool sizes = rows > 0 && rows < (1ll << 31) && widths_ok(c, hidden);
  const Plan plan = sizes ? plan_of(rows, c, hidden, precise) : Plan();
  const int wanted = (dx != nullptr ? kDx : 0) | (dw_in != nullptr ? kDwIn : 0) | (dw_out != nullptr ? kDwOut : 0);
  FfnWs w = {};
  KFB_TRY(check("feed_forward_bwd", workspace, workspace_bytes,
                sizes && wanted != 0 ? carve_gradient(w, nullptr, rows, c, hidden, precise, plan, wanted) : 0, rows, c, hidden, dtype,
                bits(dy) | bits(x) | bits(w_in) | bits(w_out) | bits(dx) | bits(dw_in) | bits(dw_out)));
  if (wanted == 0) return KFB_OK;
  carve_gradient(w, workspace, rows, c, hidden, precise, plan, wanted);
  if (nothing_kept(rows, c, hidden, precise)) {
    const int r = static_cast<int>(rows), planes = ffn_weights_planes(rows, hidden);
    if (dx != nullptr) KFB_TRY(launch_ffn_rows(s, x, dy, w_in, w_out, dx, nullptr, nullptr, r, c, hidden));
    if (dw_in == nullptr && dw_out == nullptr) return KFB_OK;
    KFB_TRY(launch_ffn_weights(s, x, dy, w_in, w_out, w.pl_in, w.pl_out, r, hidden));
    PlaneSum sums[2];
    int n = 0;
    if (dw_in != nullptr) sums[n++] = {w.pl_in, wi_n, planes, dw_in, grad_dtype == KFB_FP32, wi_n};
    if (dw_out != nullptr) sums[n++] = {w.pl_out, wo_n, planes, dw_out, grad_dtype == KFB_FP32, wo_n};
    KFB_TRY(launch_sum_planes(s, sums, n));
    return KFB_OK;
  }
  if (precise) {
    KFB_TRY(launch_split_planes(s, static_cast<const float*>(w_in), w.wi3, wi_n, wi_n));
    KFB_TRY(launch_split_planes(s, static_cast<const float*>(w_out), w.wo3, wo_n, wo_n));
  }
  const void *wi = precise ? w.wi3 : w_in, *wo = precise ? w.wo3 : w_out;
  const bool one = plan.one, sums_by_pair = plan.sums_by_pair, dx_here = plan.dx_here;
  const long long piece = plan.piece;
  const int most_in = plan.in, most_out = plan.out, dx_planes = plan.dx;
  const int grad_fp32 = grad_dtype == KFB_FP32;
  const bool single = rows <= piece;
  PlaneSum sums[3];
  int n_sums = 0;
  bool transposed = false;
  for (long long r0 = 0; r0 < rows; r0 += piece) {
    const long long r = rows - r0 < piece ? rows - r0 : piece;
    const int m = static_cast<int>(r), add = r0 > 0;
    const void *xr = static_cast<const char*>(x) + r0 * c * size, *dr = static_cast<const char*>(dy) + r0 * c * size;
    if (precise) {
      KFB_TRY(launch_split_planes(s, static_cast<const float*>(xr), w.x3, r * c, r * c));
      KFB_TRY(launch_split_planes(s, static_cast<const float*>(dr), w.dy3, r * c, r * c));
      xr = w.x3;
      dr = w.dy3;
    }
    const MatOperand mx = {xr, c, 0, r * c}, md = {dr, c, 0, r * c}, mh = {w.h, hidden, 0, r * hidden}, mg = {w.dab, 2ll * hidden, 0, r * 2 * hidden};
    auto across = [](MatOperand o) {
      o.by_k = 1;
      return o;
    };
    const bool rows_too = dx != nullptr && dx_with_hidden(m, c, hidden, one);
    void* dxr = static_cast<char*>(dx) + r0 * c * size;
    if (rows_too) {
      const bool keep = dw_in != nullptr || dw_out != nullptr;
      KFB_TRY(launch_ffn_rows(s, xr, dr, wi, wo, dxr, keep ? w.h : nullptr, keep ? w.dab : nullptr, m, c, hidden));
    } else if (one) {
      KFB_TRY(launch_ffn_hidden(s, xr, dr, wi, wo, w.h, w.dab, m, c, hidden));
    } else {
      const MatmulArgs both[2] = {{mx, {wi, c, 0, wi_n}, m, 2 * hidden, c, w.u, 2ll * hidden, 1, 1, 0, 0, precise},
                                  {md, {wo, hidden, 1, wo_n}, m, hidden, c, w.dh, hidden, 1, 1, 0, 0, precise}};
      KFB_TRY(launch_matmuls(s, both, 2, "feed_forward_in"));
      KFB_TRY(launch_hidden(s, w, true, r, hidden, precise));
    }
    MatmulArgs list[3];
    int n = 0;
    if (dx != nullptr && !rows_too) {
      if (dx_here) {
        if (dx_planes > 1) {
          list[n++] = {mg, {wi, c, 1, wi_n}, m, c, 2ll * hidden, w.pl_dx, c, 1, dx_planes, r * c, 0, precise};
          sums[n_sums++] = {w.pl_dx, r * c, dx_planes, dxr, precise, r * c};
        } else {
          list[n++] = {mg, {wi, c, 1, wi_n}, m, c, 2ll * hidden, dxr, c, precise, 1, 0, 0, precise};
        }
      } else {
        if (!transposed) KFB_TRY(launch_transpose(s, w_in, w.wi_t, 2 * hidden, c));
        transposed = true;
        KFB_TRY(product(s, w.dab, w.wi_t, dxr, r, c, 2 * hidden, "feed_forward_dx"));
      }
    }
    if (sums_by_pair) {
      if (dw_in != nullptr || dw_out != nullptr)
        KFB_TRY(launch_ffn_sums(s, w.dab, xr, w.h, dr, w.pl_in, w.pl_out, most_in, add, m, hidden));
    } else {
      // (one piece of the rows, of the contraction too: straight into the gradient)
      if (dw_in != nullptr) {
        if (single && most_in == 1) list[n++] = {across(mg), across(mx), 2 * hidden, c, r, dw_in, c, grad_fp32, 1, 0, 0, precise};
        else list[n++] = {across(mg), across(mx), 2 * hidden, c, r, w.pl_in, c, 1, pieces_of(cdiv(m, 64), most_in), wi_n, add, precise};
      }
      if (dw_out != nullptr) {
        if (single && most_out == 1) list[n++] = {across(md), across(mh), c, hidden, r, dw_out, hidden, grad_fp32, 1, 0, 0, precise};
        else list[n++] = {across(md), across(mh), c, hidden, r, w.pl_out, hidden, 1, pieces_of(cdiv(m, 64), most_out), wo_n, add, precise};
      }
    }
    if (n > 0) KFB_TRY(launch_matmuls(s, list, n, "feed_forward_products"));
  }
  if (dw_in != nullptr && (sums_by_pair || !single || most_in > 1)) sums[n_sums++] = {w.pl_in, wi_n, most_in, dw_in, grad_fp32, wi_n};
  if (dw_out != nullptr && (sums_by_pair || !single || most_out > 1)) sums[n_sums++] = {w.pl_out, wo_n, most_out, dw_out, grad_fp32, wo_n};
  return n_sums > 0 ? launch_sum_planes(s, sums, n_sums) : KFB_OK;
}

}  // extern "C"
