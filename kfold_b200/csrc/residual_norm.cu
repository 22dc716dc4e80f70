// The residual stream between two blocks:  r = scale x + sigmoid(gate) u,  y = m LayerNorm(r) + v  with (m, v) = (weight, bias) of the channels or
// (sigmoid(g), v) of gate rows that the samples of a complex share, and r kept in 8 bits beside (row_teams.cuh).
//
// What bounds it: x and u in, r and y out, HBM.  One pass: a team of lanes holds a row in registers, adds, rounds to the stream's type, and takes mean
// and variance of what it stored (residual_norm.cuh: how rows are walked and come in).  In bf16 unless said, graph replays:
//   48 x 384 rows of 768 channels, shared gates, adaptive norm, kept in 8 bits    27 us, 4.7 TB/s
//   the same rows, float32 stream, gates of their own                             48 us, 5.3 TB/s
//   384 x 384 rows of 128 channels, affine norm, kept in 8 bits                   32 us, 5.4 TB/s
//   48 x 384 rows of 768 float32 channels, gates of their own                     101 us, 3.9 TB/s; shared 60 us, 3.8
#include <mutex>

#include "ops_common.cuh"
#include "residual_norm.cuh"

namespace kfb {
namespace {

struct Params {
  const void *x, *u, *gate, *gate_shift;
  const float *scale, *weight, *bias;
  long long gate_ld, gate_shift_ld;
  void *r, *y;
  uint8_t *kept, *kept_e;
  RowPlan plan;
  int c, norm;
  float eps;
  float nothing;                       // -0, which the compiler does not know: a product with it added stays apart from the sum that follows
  int slots, s_u, s_gate, s_g;         // slots of a stage, and the first of each tensor (x: 0)
};

// r is what elementary float32 operations give, bit for bit, where these are normal numbers (smaller ones are zeros here): rows kept in 8 bits are whole numbers, and where a sum lies near a border between two of them, whoever computes it again
// should find the same one.  (A border lies within rounding of one sum in some 400 000; the fast exponential, 2^-21, missed ten times as often.)  So expf is the exact one in this
// file, and the reciprocal is rounded correctly (reciprocal_of): division itself, with its calls for denormals, made
// 48 x 384 rows of 768 channels 31.5 us where they are 27.  Gates below 10^-38 are nothing.
__device__ __forceinline__ float gate_of(float a) {
  const float w = 1.f + expf(-a);
  return w > 1e38f ? 0.f : reciprocal_of(w);
}

template <typename TS, typename TC, int P, bool OWN>
constexpr int depth() { return ring_depth(P * 8 * (sizeof(TS) + (OWN ? 4 : 1) * sizeof(TC)), OWN ? 3 : 2); }

template <typename TS, typename TC, int LANES, int P, bool VEC, int GATES>
__global__ void __launch_bounds__(kRowThreads) residual_norm_kernel(const Params p) {
  constexpr bool OWN = GATES != kSharedGates, kVectors = GATES != kOwnAdaptive;
  constexpr int kDepth = depth<TS, TC, P, OWN>(), kC = sizeof(TC) / 2;
  constexpr int kStep = LANES * kPiece;      // channels from a lane's piece to its next
  extern __shared__ uint4 ring_memory[];
  grid_dependency_enter();
  const int warp = threadIdx.x / 32, ch = threadIdx.x % LANES * (VEC ? kPiece : 1), team = threadIdx.x % 32 / LANES;
  const float inv_c = 1.0f / static_cast<float>(p.c);
  const TS* x = static_cast<const TS*>(p.x) + ch;
  const TC *u = static_cast<const TC*>(p.u) + ch, *gate = static_cast<const TC*>(p.gate) + ch, *gs = static_cast<const TC*>(p.gate_shift) + ch;
  const bool has_x = p.x != nullptr, has_u = p.u != nullptr, gated = p.gate != nullptr, adaptive = GATES == kOwnAdaptive || (GATES == kSharedGates && p.gate_shift != nullptr);
  const uint4* ring = ring_memory + threadIdx.x;
  const uint32_t ring_at = ptx::smem_u32(ring);
  int inside[P];                             // channels of a piece
#pragma unroll
  for (int q = 0; q < P; ++q) inside[q] = channels_of<VEC>(p.c, ch + q * kStep);
  auto vector = [&](const float* v, int q, float other) {
    float f[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) f[i] = v != nullptr && i < inside[q] ? v[ch + q * kStep + i * channel_step<VEC>()] : other;
    return of_floats(f);
  };

  const Pairs nothing = both(p.nothing);
  Pairs m[kVectors ? P : 1], shift[kVectors ? P : 1], open[OWN ? 1 : P];
#pragma unroll
  for (int q = 0; q < P; ++q) {
    if (kVectors) m[kVectors ? q : 0] = vector(p.weight, q, 1.f), shift[kVectors ? q : 0] = vector(p.bias, q, 0.f);
    if (!OWN) open[OWN ? 0 : q] = both(1.f);
  }

  const unsigned step = gridDim.x * (kRowThreads / 32);
  Walk<LANES, OWN> here, ahead;
  here.set = blockIdx.x * (kRowThreads / 32) + warp;
  if (here.set < p.plan.sets) here.enter(p.plan, team);
  ahead = here;
  auto fetch = [&](int stage) {
    if (ahead.set < p.plan.sets) {
      const long long o = static_cast<long long>(ahead.row) * p.c;
      const uint32_t s = ring_at + stage * p.slots * kRowThreads * 16;
      bool there[P];
#pragma unroll
      for (int q = 0; q < P; ++q) there[q] = ahead.left > 0 && inside[q] > 0;
      if (has_x) ring_copy<TS, P, kStep>(s, x + o, there);
      if (has_u) ring_copy<TC, P, kStep>(s + p.s_u * kRowThreads * 16, u + o, there);
      if (OWN && gated) ring_copy<TC, P, kStep>(s + p.s_gate * kRowThreads * 16, gate + ahead.row * p.gate_ld, there);
      if (OWN && adaptive) {
        ring_copy<TC, P, kStep>(s + p.s_g * kRowThreads * 16, gs + ahead.row * p.gate_shift_ld, there);
        ring_copy<TC, P, kStep>(s + (p.s_g + P * kC) * kRowThreads * 16, gs + ahead.row * p.gate_shift_ld + p.c, there);
      }
      ahead.next(p.plan, team, step);
    }
    copy_async_done();
  };
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) fetch(i);
  }
  int stage = 0;
  while (here.set < p.plan.sets) {
    if constexpr (VEC) {
      fetch(stage == 0 ? kDepth - 1 : stage - 1);
      copy_async_wait<kDepth - 1>();
    } else {
      ahead.next(p.plan, team, step);
      if (ahead.set < p.plan.sets && ahead.left > 0) {
        const int lane = threadIdx.x % 32;
        const long long o = static_cast<long long>(ahead.row) * p.c - ch;
        if (has_x) prefetch_row(x + o, p.c, lane);
        if (has_u) prefetch_row(u + o, p.c, lane);
        if (OWN && gated) prefetch_row(gate - ch + ahead.row * p.gate_ld, p.c, lane);
        if (OWN && adaptive) prefetch_row(gs - ch + ahead.row * p.gate_shift_ld, 2 * p.c, lane);
      }
    }
    const uint4* s = ring + stage * p.slots * kRowThreads;
    const long long o = static_cast<long long>(here.row) * p.c + ch;
    int k[P];                                // channels that are there
#pragma unroll
    for (int q = 0; q < P; ++q) k[q] = here.left > 0 ? inside[q] : 0;
    // (from: this lane's first piece)
    auto take = [&](auto tag, int slot, const auto* from, int q) {
      using E = decltype(tag);
      if constexpr (VEC) return ring_take<E>(s + (slot + q * (static_cast<int>(sizeof(E)) / 2)) * kRowThreads);
      else return load_piece<E, VEC>(from + q * kStep, k[q]);
    };
    if (!OWN && here.at == 0) {
      const unsigned gate_row = here.gate_row(p.plan);
      if (gated) {
#pragma unroll
        for (int q = 0; q < P; ++q)
          open[OWN ? 0 : q] = each(load_piece<TC, VEC>(gate + gate_row * p.gate_ld + q * kStep, k[q]), gate_of);
      }
      if (adaptive) {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          m[kVectors ? q : 0] = each(load_piece<TC, VEC>(gs + gate_row * p.gate_shift_ld + q * kStep, k[q]), [](float a) { return open_of(gate_at<TC>(a)); });
          shift[kVectors ? q : 0] = load_piece<TC, VEC>(gs + gate_row * p.gate_shift_ld + p.c + q * kStep, k[q]);
        }
      }
    }
    // (a question that is the same for all pieces is asked once: the pieces' instructions then lie side by side)
    Pairs r[P];
    if (has_x) {
#pragma unroll
      for (int q = 0; q < P; ++q) r[q] = take(TS{}, 0, x + (o - ch), q);
      if (p.scale != nullptr) {
#pragma unroll
        for (int q = 0; q < P; ++q) r[q] = fma(r[q], vector(p.scale, q, 0.f), nothing);
      }
    } else {
#pragma unroll
      for (int q = 0; q < P; ++q) r[q] = both(0.f);
    }
    if (has_u) {
      if (OWN && gated) {
#pragma unroll
        for (int q = 0; q < P; ++q)
          r[q] = add(r[q], fma(each(take(TC{}, p.s_gate, gate + here.row * p.gate_ld, q), gate_of), take(TC{}, p.s_u, u + (o - ch), q), nothing));
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const Pairs t = take(TC{}, p.s_u, u + (o - ch), q);
          r[q] = add(r[q], OWN ? t : fma(open[OWN ? 0 : q], t, nothing));
        }
      }
    }
    // as it is stored
    TS* to = static_cast<TS*>(p.r) + o;
    uint32_t top[P];
    if constexpr (std::is_same<TS, __nv_bfloat16>::value) {
      uint4 w[P];
#pragma unroll
      for (int q = 0; q < P; ++q) {
        w[q] = to_bf16(r[q]);
        r[q] = of_bf16(w[q]);
        top[q] = top_of(w[q]);
      }
      if constexpr (VEC) {
        if (p.r != nullptr) {
#pragma unroll
          for (int q = 0; q < P; ++q)
            if (k[q] > 0) *reinterpret_cast<uint4*>(to + q * kStep) = w[q];
        }
      }
    }
    if (!(VEC && std::is_same<TS, __nv_bfloat16>::value) && p.r != nullptr) {
#pragma unroll
      for (int q = 0; q < P; ++q) store_piece<VEC>(to + q * kStep, r[q], k[q]);
    }
    if (p.kept != nullptr) {
      uint8_t *bytes = p.kept + o, *e = p.kept_e + static_cast<long long>(here.row) * groups8(p.c);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        if constexpr (!std::is_same<TS, __nv_bfloat16>::value) top[q] = top_of(r[q]);
        store_piece8<VEC>(bytes + q * kStep, e + (ch + q * kStep) / kGroup8, r[q], top[q], k[q], threadIdx.x % 32);
      }
    }
    if (p.norm != kNoNorm) {
      Pairs sum = r[0];
#pragma unroll
      for (int q = 1; q < P; ++q) sum = add(sum, r[q]);
      float t[1] = {total(sum)};
      team_sum<LANES>(t);
      const float mean = t[0] * inv_c;
      sum = both(0.f);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        r[q] = add(r[q], both(inside[q] > 0 ? -mean : 0.f));      // (nothing stays nothing)
        if constexpr (!VEC) {
#pragma unroll
          for (int i = 0; i < kPiece; ++i)
            if (i >= inside[q]) r[q].v[i / 2] = i & 1 ? ptx::pack2(r[q].get(i - 1), 0.f) : ptx::pack2(0.f, 0.f);
        }
        sum = fma(r[q], r[q], sum);
      }
      t[0] = total(sum);
      team_sum<LANES>(t);
      const Pairs rstd = both(rsqrtf(fmaf(t[0], inv_c, p.eps)));
      if (OWN && adaptive) {
#pragma unroll
        for (int q = 0; q < P; ++q)
          r[q] = fma(mul(r[q], rstd), each(take(TC{}, p.s_g, gs + here.row * p.gate_shift_ld, q), [](float a) { return open_of(gate_at<TC>(a)); }),
                     take(TC{}, p.s_g + P * kC, gs + here.row * p.gate_shift_ld + p.c, q));
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) r[q] = fma(mul(r[q], rstd), m[kVectors ? q : 0], shift[kVectors ? q : 0]);
      }
      TC* y = static_cast<TC*>(p.y) + o;
#pragma unroll
      for (int q = 0; q < P; ++q) store_piece<VEC>(y + q * kStep, r[q], k[q]);
    }
    here.next(p.plan, team, step);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
  }
}

template <typename TS, typename TC, int LANES, int P, bool VEC, int GATES>
int launch(cudaStream_t stream, Params p, long long rows, int samples, int l) {
  constexpr bool OWN = GATES != kSharedGates;
  constexpr auto kernel = residual_norm_kernel<TS, TC, LANES, P, VEC, GATES>;
  constexpr int kWarps = kRowThreads / 32, kTeams = 32 / LANES, kMostBlocks = 8;
  static std::once_flag once;
  static int held = 1;
  std::call_once(once, [&] {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, kRowThreads, 0) != cudaSuccess) cudaGetLastError();
    held = held < 1 ? 1 : held > kMostBlocks ? kMostBlocks : held;
  });
  constexpr int kS = P * sizeof(TS) / 2, kC = P * sizeof(TC) / 2;        // slots of a tensor
  p.slots = p.x != nullptr ? kS : 0;
  p.s_u = p.slots;
  p.slots += p.u != nullptr ? kC : 0;
  p.s_gate = p.slots;
  p.slots += OWN && p.gate != nullptr ? kC : 0;
  p.s_g = p.slots;
  p.slots += OWN && p.gate_shift != nullptr ? 2 * kC : 0;
  const int smem = VEC ? depth<TS, TC, P, OWN>() * p.slots * kRowThreads * 16 : 0;
  if (VEC) KFB_TRY(allow_smem<kernel>(kMostRing));
  const int room = smem > 0 ? kMostRing / smem : held, blocks_per_sm = held < room ? held : room < 1 ? 1 : room;
  const long long most = static_cast<long long>(sm_count()) * blocks_per_sm;
  p.plan = row_plan(rows, samples, l, most * kWarps * kTeams, kTeams, 0);
  const long long want = (p.plan.sets + kWarps - 1) / kWarps;
  LaunchScope scope(stream, "residual_norm");
  return launch_kernel(stream, kernel, static_cast<unsigned>(want < most ? want : most), kRowThreads, smem, p);
}

template <typename TS, typename TC, int LANES, int P, bool VEC>
int launch_own(cudaStream_t stream, const Params& p, long long rows, int samples, int l) {
  if (samples > 1) return launch<TS, TC, LANES, P, VEC, kSharedGates>(stream, p, rows, samples, l);
  return p.norm == kAdaptiveNorm ? launch<TS, TC, LANES, P, VEC, kOwnAdaptive>(stream, p, rows, samples, l)
                                 : launch<TS, TC, LANES, P, VEC, kOwnGates>(stream, p, rows, samples, l);
}

template <typename TS, typename TC>
int dispatch(cudaStream_t stream, const Params& p, long long rows, int samples, int l) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.u) | reinterpret_cast<uintptr_t>(p.gate) |
                       reinterpret_cast<uintptr_t>(p.gate_shift) | reinterpret_cast<uintptr_t>(p.r) | reinterpret_cast<uintptr_t>(p.y) |
                       static_cast<uintptr_t>((p.gate_ld | p.gate_shift_ld) * sizeof(TC)) | (reinterpret_cast<uintptr_t>(p.kept) & 7);
#define KFB_CALL(LANES, P, VEC) launch_own<TS, TC, LANES, P, VEC>(stream, p, rows, samples, l)
  KFB_ROW_SHAPES(p.c, p.c % 8 == 0 && (at & 15) == 0, KFB_CALL);
#undef KFB_CALL
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
  p.nothing = -0.f;
  cudaStream_t s = as_stream(stream);
  if (stream_dtype == KFB_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(s, p, rows, each, l);
  return compute_dtype == KFB_BF16 ? dispatch<float, __nv_bfloat16>(s, p, rows, each, l) : dispatch<float, float>(s, p, rows, each, l);
}

}  // extern "C"
