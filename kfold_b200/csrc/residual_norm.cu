// The residual stream between two blocks:  r = scale x + sigmoid(gate) u,  y = m LayerNorm(r) + v  with (m, v) = (weight, bias) of the channels or
// (sigmoid(g), v) of gate rows that the samples of a complex share, and r kept in 8 bits beside (row_teams.cuh).
//
// What bounds it: x and u in, r and y out, HBM.  One pass: a team of lanes holds a row in registers, adds, rounds to the stream's type, and takes mean
// and variance of what it stored (residual_norm.cuh: how rows are walked and come in).
#include <mutex>
#include <type_traits>

#include "ops_common.cuh"
#include "residual_norm.cuh"

namespace kfb {
namespace {

constexpr int kDepth = 4;              // rows on their way for a team, the one in work among them

struct Params {
  const void *x, *u, *gate, *gate_shift;
  const float *scale, *weight, *bias;
  long long gate_ld, gate_shift_ld;
  void *r, *y;
  uint8_t *kept, *kept_e;
  RowPlan plan;
  int c, norm;
  float eps;
  int slots, s_u, s_gate, s_g;         // slots of a stage, and the first of each tensor (x: 0)
};

template <typename T>
__device__ __forceinline__ float as_stored(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(__float2bfloat16_rn(v));
  else return v;
}

template <typename TS, typename TC, int LANES, bool VEC, bool OWN>
__global__ void __launch_bounds__(Teams<LANES>::kThreads) residual_norm_kernel(const Params p) {
  using T = Teams<LANES>;
  constexpr int N = kPiece;
  __shared__ float room[2][T::kGroups][T::kWarps][1];
  extern __shared__ uint4 ring_memory[];
  grid_dependency_enter();
  const int group = threadIdx.x / T::kGroupLanes, sub = threadIdx.x % LANES, team = threadIdx.x % T::kGroupLanes / LANES;
  const int ch = sub * N, n = min(max(p.c - ch, 0), N);
  const float inv_c = 1.0f / static_cast<float>(p.c);
  const TS* x = static_cast<const TS*>(p.x);
  const TC *u = static_cast<const TC*>(p.u), *gate = static_cast<const TC*>(p.gate), *gs = static_cast<const TC*>(p.gate_shift);
  uint4* ring = ring_memory + threadIdx.x;

  float m[N], shift[N], open[OWN ? 1 : N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = p.weight != nullptr && i < n ? p.weight[ch + i] : 1.f;
    shift[i] = p.bias != nullptr && i < n ? p.bias[ch + i] : 0.f;
    if (!OWN) open[i] = 1.f;
  }

  const unsigned step = gridDim.x * T::kGroups;
  Walk<LANES, OWN> here, ahead;
  here.set = blockIdx.x * T::kGroups + group;
  if (here.set < p.plan.sets) here.enter(p.plan, team);
  ahead = here;
  auto fetch = [&](int stage) {
    if (ahead.set < p.plan.sets) {
      uint4* q = ring + stage * p.slots * T::kThreads;
      const bool there = ahead.left > 0 && n > 0;
      const long long o = static_cast<long long>(ahead.row) * p.c + ch;
      if (x != nullptr) ring_copy<TS, VEC>(q, T::kThreads, x + o, there);
      if (u != nullptr) ring_copy<TC, VEC>(q + p.s_u * T::kThreads, T::kThreads, u + o, there);
      if (OWN && gate != nullptr) ring_copy<TC, VEC>(q + p.s_gate * T::kThreads, T::kThreads, gate + ahead.row * p.gate_ld + ch, there);
      if (OWN && gs != nullptr) {
        uint4* g = q + p.s_g * T::kThreads;
        ring_copy<TC, VEC>(g, T::kThreads, gs + ahead.row * p.gate_shift_ld + ch, there);
        ring_copy<TC, VEC>(g + sizeof(TC) / 2 * T::kThreads, T::kThreads, gs + ahead.row * p.gate_shift_ld + p.c + ch, there);
      }
      ahead.next(p.plan, team, step);
    }
    copy_async_done();
  };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) fetch(i);
  }
  int turn = 0, stage = 0;
  while (here.set < p.plan.sets) {
    if constexpr (VEC) {
      fetch(stage == 0 ? kDepth - 1 : stage - 1);
      copy_async_wait<kDepth - 1>();
    }
    const int k = here.left > 0 ? n : 0;
    const uint4* q = ring + stage * p.slots * T::kThreads;
    const long long o = static_cast<long long>(here.row) * p.c + ch;
    float r[N], t[N];
    Piece<TC, VEC> raw;
    if (!OWN && here.at == 0) {
      const unsigned gate_row = here.gate_row(p.plan);
      if (gate != nullptr) {
        raw.load(gate + gate_row * p.gate_ld + ch, k);
        raw.values(t);
#pragma unroll
        for (int i = 0; i < (OWN ? 1 : N); ++i) open[i] = open_exact(t[i]);
      }
      if (gs != nullptr) {
        raw.load(gs + gate_row * p.gate_shift_ld + ch, k);
        raw.values(t);
        raw.load(gs + gate_row * p.gate_shift_ld + p.c + ch, k);
        raw.values(shift);
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = gate_at(t[i]).open;
      }
    }
    if (x != nullptr) {
      Piece<TS, VEC> x_raw;
      if constexpr (VEC) x_raw.take(q, T::kThreads);
      else x_raw.load(x + o, k);
      x_raw.values(r);
      if (p.scale != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] *= i < n ? p.scale[ch + i] : 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = 0.f;
    }
    if (u != nullptr) {
      if constexpr (VEC) raw.take(q + p.s_u * T::kThreads, T::kThreads);
      else raw.load(u + o, k);
      raw.values(t);
      if (gate == nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] += t[i];
      } else if constexpr (OWN) {
        float s[N];
        if constexpr (VEC) raw.take(q + p.s_gate * T::kThreads, T::kThreads);
        else raw.load(gate + here.row * p.gate_ld + ch, k);
        raw.values(s);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fmaf(open_exact(s[i]), t[i], r[i]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fmaf(open[i], t[i], r[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = as_stored<TS>(r[i]);
    if (p.r != nullptr) store_piece<VEC>(static_cast<TS*>(p.r) + o, r, k);
    if (p.kept != nullptr)
      store_piece8<VEC>(p.kept + o, p.kept_e + static_cast<long long>(here.row) * groups8(p.c) + ch / kGroup8, r, k, sub % (kGroup8 / N) == 0);
    if (p.norm != kNoNorm) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] += r[i];
      team_sum<LANES>(s, room, group, turn);
      const float mean = s[0] * inv_c;
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        r[i] = (VEC ? n > 0 : i < n) ? r[i] - mean : 0.f;
        s[0] = fmaf(r[i], r[i], s[0]);
      }
      team_sum<LANES>(s, room, group, turn ^ 1);
      const float rstd = rsqrtf(fmaf(s[0], inv_c, p.eps));
      if (OWN && gs != nullptr) {
        if constexpr (VEC) raw.take(q + p.s_g * T::kThreads, T::kThreads);
        else raw.load(gs + here.row * p.gate_shift_ld + ch, k);
        raw.values(t);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = r[i] * rstd * gate_at(t[i]).open;
        if constexpr (VEC) raw.take(q + (p.s_g + static_cast<int>(sizeof(TC)) / 2) * T::kThreads, T::kThreads);
        else raw.load(gs + here.row * p.gate_shift_ld + p.c + ch, k);
        raw.values(t);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] += t[i];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = fmaf(r[i] * rstd, m[i], shift[i]);
      }
      store_piece<VEC>(static_cast<TC*>(p.y) + o, r, k);
    }
    here.next(p.plan, team, step);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
  }
}

constexpr int kMostRing = 200 * 1024;

template <typename TS, typename TC, int LANES, bool VEC, bool OWN>
int launch(cudaStream_t stream, Params p, long long rows, int samples, int l) {
  using T = Teams<LANES>;
  constexpr auto kernel = residual_norm_kernel<TS, TC, LANES, VEC, OWN>;
  static std::once_flag once;
  static int held = 1;
  std::call_once(once, [&] {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, T::kThreads, 0) != cudaSuccess) cudaGetLastError();
    held = held < 1 ? 1 : held > 4 ? 4 : held;
  });
  constexpr int kS = sizeof(TS) / 2, kC = sizeof(TC) / 2;        // slots of a piece
  p.slots = p.x != nullptr ? kS : 0;
  p.s_u = p.slots;
  p.slots += p.u != nullptr ? kC : 0;
  p.s_gate = p.slots;
  p.slots += OWN && p.gate != nullptr ? kC : 0;
  p.s_g = p.slots;
  p.slots += OWN && p.gate_shift != nullptr ? 2 * kC : 0;
  const int smem = VEC ? kDepth * p.slots * T::kThreads * 16 : 0;
  if (VEC) KFB_TRY(allow_smem<kernel>(kMostRing));
  const int room = smem > 0 ? kMostRing / smem : held, blocks_per_sm = held < room ? held : room < 1 ? 1 : room;
  const long long most = static_cast<long long>(sm_count()) * blocks_per_sm, teams = T::kGroups * T::kTeams;
  p.plan = row_plan(rows, samples, l, most * teams, T::kTeams);
  const long long want = (p.plan.sets + T::kGroups - 1) / T::kGroups;
  LaunchScope scope(stream, "residual_norm");
  return launch_kernel(stream, kernel, static_cast<unsigned>(want < most ? want : most), T::kThreads, smem, p);
}

template <typename TS, typename TC, int LANES, bool VEC>
int launch_own(cudaStream_t stream, const Params& p, long long rows, int samples, int l) {
  return samples == 1 ? launch<TS, TC, LANES, VEC, true>(stream, p, rows, samples, l) : launch<TS, TC, LANES, VEC, false>(stream, p, rows, samples, l);
}

template <typename TS, typename TC>
int dispatch(cudaStream_t stream, const Params& p, long long rows, int samples, int l) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.u) | reinterpret_cast<uintptr_t>(p.gate) |
                       reinterpret_cast<uintptr_t>(p.gate_shift) | reinterpret_cast<uintptr_t>(p.r) | reinterpret_cast<uintptr_t>(p.y) |
                       static_cast<uintptr_t>((p.gate_ld | p.gate_shift_ld) * sizeof(TC)) | (reinterpret_cast<uintptr_t>(p.kept) & 7);
  if (p.c % 8 == 0 && (at & 15) == 0) {
    if (p.c <= 64) return launch_own<TS, TC, 8, true>(stream, p, rows, samples, l);
    if (p.c <= 128) return launch_own<TS, TC, 16, true>(stream, p, rows, samples, l);
    if (p.c <= 256) return launch_own<TS, TC, 32, true>(stream, p, rows, samples, l);
    if (p.c <= 512) return launch_own<TS, TC, 64, true>(stream, p, rows, samples, l);
    if (p.c <= 768) return launch_own<TS, TC, 96, true>(stream, p, rows, samples, l);
    return launch_own<TS, TC, 128, true>(stream, p, rows, samples, l);
  }
  return p.c <= 256 ? launch_own<TS, TC, 32, false>(stream, p, rows, samples, l) : launch_own<TS, TC, 128, false>(stream, p, rows, samples, l);
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
  const int each = shared ? samples : 1;
  p.c = c;
  p.norm = norm;
  p.eps = eps;
  cudaStream_t s = as_stream(stream);
  if (stream_dtype == KFB_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(s, p, rows, each, l);
  return compute_dtype == KFB_BF16 ? dispatch<float, __nv_bfloat16>(s, p, rows, each, l) : dispatch<float, float>(s, p, rows, each, l);
}

}  // extern "C"
