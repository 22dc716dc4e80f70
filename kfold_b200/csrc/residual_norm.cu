// The residual stream between two blocks:  r = scale x + sigmoid(gate) u,  y = m LayerNorm(r) + v  with (m, v) = (weight, bias) of the channels or
// (sigmoid(g), v) of gate rows that the samples of a complex share, and r kept in 8 bits beside (row_teams.cuh).
//
// What bounds it: x and u in, r and y out, HBM.  One pass: a team of lanes holds a row in registers, adds, rounds to the stream's type, and takes mean
// and variance of what it stored.  A team walks the samples that share a gate row one after the other, so that gates are read and their
// exponentials computed once for all of them; where gate rows are few, the samples are cut into pieces.  The next row's loads stand before this
// row's stores.
#include <type_traits>

#include "ops_common.cuh"
#include "residual_norm.cuh"
#include "row_teams.cuh"

namespace kfb {
namespace {

struct Params {
  const void *x, *u, *gate, *gate_shift;
  const float *scale, *weight, *bias;
  long long gate_ld, gate_shift_ld;
  void *r, *y;
  uint8_t *kept, *kept_e;
  RowShare share;
  unsigned units;        // pieces of at most `chunk` samples of a gate row, `chunks` of them each
  int chunks, chunk;
  int c, norm;
  float eps;
};

template <typename T>
__device__ __forceinline__ float as_stored(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(__float2bfloat16_rn(v));
  else return v;
}

template <typename TS, typename TC, int LANES, bool VEC>
__global__ void __launch_bounds__(Teams<LANES>::kThreads) residual_norm_kernel(const Params p) {
  using T = Teams<LANES>;
  __shared__ float room[2][T::kGroups][T::kWarps][1];
  grid_dependency_enter();
  const int group = threadIdx.x / T::kGroupLanes, sub = threadIdx.x % LANES, team = threadIdx.x % T::kGroupLanes / LANES;
  const int ch = sub * kPiece, n = min(max(p.c - ch, 0), kPiece);
  const float inv_c = 1.0f / static_cast<float>(p.c);
  const TS* x = static_cast<const TS*>(p.x);
  const TC *u = static_cast<const TC*>(p.u), *gate = static_cast<const TC*>(p.gate), *gs = static_cast<const TC*>(p.gate_shift);

  float scale[kPiece], m[kPiece], shift[kPiece], open[kPiece];
#pragma unroll
  for (int i = 0; i < kPiece; ++i) {
    scale[i] = p.scale != nullptr && i < n ? p.scale[ch + i] : 1.f;
    m[i] = p.weight != nullptr && i < n ? p.weight[ch + i] : 1.f;
    shift[i] = p.bias != nullptr && i < n ? p.bias[ch + i] : 0.f;
    open[i] = 1.f;
  }

  const unsigned sets = (p.units + T::kTeams - 1) / T::kTeams, step = gridDim.x * T::kGroups;
  unsigned set = blockIdx.x * T::kGroups + group, row = 0, cond = 0;
  int left = 0, at = 0;                       // samples of this team's piece from here on; how many the group has taken
  Piece<TS, VEC> x_raw;
  Piece<TC, VEC> u_raw, gate_raw, g_raw, v_raw;
  auto enter = [&] {
    const unsigned unit = set * T::kTeams + team;
    const bool there = unit < p.units;
    const int first = there ? static_cast<int>(unit % p.chunks) * p.chunk : 0;
    cond = there ? unit / p.chunks : 0;
    left = there ? min(p.chunk, p.share.samples - first) : 0;
    row = p.share.row(cond, first);
    const int k = left > 0 ? n : 0;
    if (gate != nullptr) gate_raw.load(gate + cond * p.gate_ld + ch, k);
    if (gs != nullptr) {
      g_raw.load(gs + cond * p.gate_shift_ld + ch, k);
      v_raw.load(gs + cond * p.gate_shift_ld + p.c + ch, k);
    }
  };
  auto fetch = [&] {
    const int k = left > 0 ? n : 0;
    const long long o = static_cast<long long>(row) * p.c + ch;
    if (x != nullptr) x_raw.load(x + o, k);
    if (u != nullptr) u_raw.load(u + o, k);
  };
  if (set < sets) {
    enter();
    fetch();
  }
  int turn = 0;
  while (set < sets) {
    float r[kPiece], t[kPiece];
    if (x != nullptr) {
      x_raw.values(r);
    } else {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) r[i] = 0.f;
    }
    if (at == 0) {
      if (gate != nullptr) {
        gate_raw.values(t);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) open[i] = open_exact(t[i]);
      }
      if (gs != nullptr) {
        g_raw.values(t);
        v_raw.values(shift);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) m[i] = gate_at(t[i]).open;
      }
    }
    if (p.scale != nullptr) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) r[i] *= scale[i];
    }
    if (u != nullptr) {
      u_raw.values(t);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) r[i] = fmaf(open[i], t[i], r[i]);
    }
    const int here = left > 0 ? n : 0;
    const unsigned this_row = row;
    if (++at == p.chunk) {
      at = 0;
      set += step;
      if (set < sets) enter();
    } else {
      --left;
      row += p.share.l;
    }
    if (set < sets) fetch();

    const long long o = static_cast<long long>(this_row) * p.c + ch;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) r[i] = as_stored<TS>(r[i]);
    if (p.r != nullptr) store_piece<VEC>(static_cast<TS*>(p.r) + o, r, here);
    if (p.kept != nullptr) {
      const int groups = groups8(p.c);
      store_piece8<VEC>(p.kept + o, p.kept_e + static_cast<long long>(this_row) * groups + ch / kGroup8, r, here, sub % (kGroup8 / kPiece) == 0);
    }
    if (p.norm != kNoNorm) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < kPiece; ++i) s[0] += r[i];
      team_sum<LANES>(s, room, group, turn);
      turn ^= 1;
      const float mean = s[0] * inv_c;
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        r[i] = (VEC ? n > 0 : i < n) ? r[i] - mean : 0.f;
        s[0] = fmaf(r[i], r[i], s[0]);
      }
      team_sum<LANES>(s, room, group, turn);
      turn ^= 1;
      const float rstd = rsqrtf(fmaf(s[0], inv_c, p.eps));
#pragma unroll
      for (int i = 0; i < kPiece; ++i) r[i] = fmaf(r[i] * rstd, m[i], shift[i]);
      store_piece<VEC>(static_cast<TC*>(p.y) + o, r, here);
    }
  }
}

template <typename TS, typename TC, int LANES, bool VEC>
int launch(cudaStream_t stream, Params p) {
  using T = Teams<LANES>;
  auto kernel = residual_norm_kernel<TS, TC, LANES, VEC>;
  static std::once_flag once;
  static int held = 1;
  std::call_once(once, [&] {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, T::kThreads, 0) != cudaSuccess) cudaGetLastError();
    held = held < 1 ? 1 : held > 4 ? 4 : held;
  });
  // as many pieces of a gate row's samples as give every team one
  const unsigned most = static_cast<unsigned>(sm_count()) * held, teams = T::kGroups * T::kTeams;
  p.chunks = 1;
  if (p.share.samples > 1 && p.share.cond_rows < most * teams) {
    const unsigned want = (most * teams + p.share.cond_rows - 1) / p.share.cond_rows;
    p.chunks = static_cast<int>(want < static_cast<unsigned>(p.share.samples) ? want : p.share.samples);
  }
  p.chunk = cdiv(p.share.samples, p.chunks);
  p.chunks = cdiv(p.share.samples, p.chunk);
  p.units = p.share.cond_rows * p.chunks;
  const unsigned want = (p.units + teams - 1) / teams;
  LaunchScope scope(stream, "residual_norm");
  return launch_kernel(stream, kernel, want < most ? want : most, T::kThreads, 0, p);
}

template <typename TS, typename TC>
int dispatch(cudaStream_t stream, const Params& p) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.u) | reinterpret_cast<uintptr_t>(p.gate) |
                       reinterpret_cast<uintptr_t>(p.gate_shift) | reinterpret_cast<uintptr_t>(p.r) | reinterpret_cast<uintptr_t>(p.y) |
                       static_cast<uintptr_t>((p.gate_ld | p.gate_shift_ld) * sizeof(TC)) | (reinterpret_cast<uintptr_t>(p.kept) & 7);
  if (p.c % 8 == 0 && (at & 15) == 0) {
    if (p.c <= 64) return launch<TS, TC, 8, true>(stream, p);
    if (p.c <= 128) return launch<TS, TC, 16, true>(stream, p);
    if (p.c <= 256) return launch<TS, TC, 32, true>(stream, p);
    if (p.c <= 512) return launch<TS, TC, 64, true>(stream, p);
    if (p.c <= 768) return launch<TS, TC, 96, true>(stream, p);
    return launch<TS, TC, 128, true>(stream, p);
  }
  return p.c <= 256 ? launch<TS, TC, 32, false>(stream, p) : launch<TS, TC, 128, false>(stream, p);
}

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API int kfb_residual_norm_fwd(const void* x, const void* u, const void* gate, long long gate_ld, const float* scale, const float* weight,
                                  const float* bias, const void* gate_shift, long long gate_shift_ld, void* r, void* y, void* kept,
                                  void* kept_exponents, long long rows, int c, int samples, int l, float eps, int norm, int stream_dtype,
                                  int compute_dtype, void* stream) {
  KFB_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && c > 0 && samples > 0 && l > 0 && rows % (static_cast<long long>(samples) * l) == 0,
                "residual_norm: rows %lld of %d channels, %d samples of %d tokens", rows, c, samples, l);
  if (c > 1024) {
    set_error("residual_norm: channel count %d above 1024 is not supported", c);
    return KFB_ERR_UNSUPPORTED;
  }
  KFB_CHECK_ARG((stream_dtype == KFB_BF16 && compute_dtype == KFB_BF16) || (stream_dtype == KFB_FP32 && (compute_dtype == KFB_BF16 || compute_dtype == KFB_FP32)),
                "residual_norm: dtypes %d and %d", stream_dtype, compute_dtype);
  KFB_CHECK_ARG(norm >= kNoNorm && norm <= kAdaptiveNorm && (norm == kAdaptiveNorm) == (gate_shift != nullptr) &&
                    (norm == kAffineNorm || (weight == nullptr && bias == nullptr)), "residual_norm: norm %d with other parameters", norm);
  KFB_CHECK_ARG((gate == nullptr || (u != nullptr && gate_ld >= c)) && (gate_shift == nullptr || gate_shift_ld >= 2ll * c),
                "residual_norm: gate rows %lld and %lld apart", gate_ld, gate_shift_ld);
  if (rows == 0) return KFB_OK;
  KFB_CHECK_ARG((x != nullptr || u != nullptr) && (norm == kNoNorm || y != nullptr) && (kept == nullptr) == (kept_exponents == nullptr), "residual_norm: null tensor");
  KFB_CHECK_ARG(r != nullptr || (u == nullptr && scale == nullptr), "residual_norm: no place for the sum");
  Params p = {};
  p.x = x;
  p.u = u;
  p.gate = gate;
  p.gate_shift = gate_shift;
  p.scale = scale;
  p.weight = weight;
  p.bias = bias;
  p.gate_ld = gate != nullptr ? gate_ld : 0;
  p.gate_shift_ld = gate_shift != nullptr ? gate_shift_ld : 0;
  p.r = r;
  p.y = norm == kNoNorm ? nullptr : y;
  p.kept = static_cast<uint8_t*>(kept);
  p.kept_e = static_cast<uint8_t*>(kept_exponents);
  const bool shared = samples > 1 && (gate != nullptr || gate_shift != nullptr);
  p.share = {static_cast<unsigned>(shared ? rows / samples : rows), static_cast<unsigned>(l), shared ? samples : 1};
  p.c = c;
  p.norm = norm;
  p.eps = eps;
  cudaStream_t s = as_stream(stream);
  if (stream_dtype == KFB_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(s, p);
  return compute_dtype == KFB_BF16 ? dispatch<float, __nv_bfloat16>(s, p) : dispatch<float, float>(s, p);
}

}  // extern "C"
