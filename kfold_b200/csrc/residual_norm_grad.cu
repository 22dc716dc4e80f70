// The gradient of residual_norm.cu.  With z = (r - mean) rstd of the stored r, m the factor of the norm and s = sigmoid(gate):
//   g = m dy,  t = dr + rstd (g - mean(g) - z mean(g z)),  dx = scale t,  du = s t,
//   dgate = s (1 - s) sum(t u),  d gate_shift = [m (1 - m) sum(dy z) | sum(dy)]  over the samples that share the row,
//   dweight = sum(dy z),  dbias = sum(dy),  dscale = sum(t x)  over all rows.
//
// What bounds it: dr, dy, r and u in, dx and du out, HBM.  Row statistics come from r again.  r, u and x may be the tensors or rows kept in 8 bits
// (row_teams.cuh), which are taken apart in registers.
// Split: as in residual_norm.cu a team of lanes holds a row and walks the samples that share its gates, their sums in registers; where gate rows are
// few the teams of a block take the samples of one row between them and meet in shared memory.  Sums over all rows stay in registers from row to
// row; a block leaves a row of partial sums, which a second kernel adds in the blocks' order.  No atomics: the order hangs on the sizes alone.
#include "ops_common.cuh"
#include "residual_norm.cuh"
#include "row_teams.cuh"

namespace kfb {
namespace {

struct GradParams {
  const void *dr, *dy, *r, *u, *x, *gate, *gate_shift;
  const uint8_t *r_e, *u_e, *x_e;      // exponents of those that are kept in 8 bits
  const float *scale, *weight;
  long long gate_ld, gate_shift_ld;
  void *dx, *du, *dgate, *dgate_shift;
  float* partial;                      // [block][3][c]: sums of dy z, dy, t x
  RowShare share;
  unsigned sets;                       // of gate rows that a group (split: a block) takes at a time
  int chunk, split;
  int c, norm;
  float eps;
};

// OWN: a row has gates of its own.
template <typename TS, typename TC, int LANES, bool VEC, bool OWN>
__global__ void __launch_bounds__(Teams<LANES>::kThreads) residual_norm_grad_kernel(const GradParams p) {
  using T = Teams<LANES>;
  constexpr int N = kPiece;
  __shared__ float room[2][T::kGroups][T::kWarps][2];
  __shared__ float4 s_sum[OWN ? 1 : 3][T::kThreads * 2];
  grid_dependency_enter();
  const int group = threadIdx.x / T::kGroupLanes, sub = threadIdx.x % LANES, team = threadIdx.x % T::kGroupLanes / LANES;
  const int ch = sub * N, n = min(max(p.c - ch, 0), N), groups = groups8(p.c);
  const float inv_c = 1.0f / static_cast<float>(p.c);
  const TS *dr = static_cast<const TS*>(p.dr), *r = static_cast<const TS*>(p.r), *x = static_cast<const TS*>(p.x);
  const TC *dy = static_cast<const TC*>(p.dy), *u = static_cast<const TC*>(p.u), *gate = static_cast<const TC*>(p.gate),
           *gs = static_cast<const TC*>(p.gate_shift);
  const bool adaptive = p.norm == kAdaptiveNorm;

  float m[N], open[N], a0[N], a1[N], a2[N], a3[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = p.weight != nullptr && i < n ? p.weight[ch + i] : 1.f;
    open[i] = 1.f;
    a0[i] = a1[i] = a2[i] = a3[i] = 0.f;
  }

  const unsigned step = p.split ? gridDim.x : gridDim.x * T::kGroups;
  unsigned set = p.split ? blockIdx.x : blockIdx.x * T::kGroups + group, row = 0, cond = 0;
  int left = 0, at = 0;
  bool there = false;
  Piece<TS, VEC> dr_raw, r_raw, x_raw;
  Piece<TC, VEC> dy_raw, u_raw, gate_raw, g_raw;
  auto enter = [&] {
    const unsigned unit = set * T::kTeams + team;
    there = unit < p.share.cond_rows;
    const int first = p.split ? group * p.chunk : 0;
    cond = there ? unit : 0;
    left = there ? min(p.chunk, p.share.samples - first) : 0;
    row = OWN ? cond : p.share.row(cond, first);
  };
  auto gates = [&] {
    const int k = there ? n : 0;
    if (gate != nullptr) gate_raw.load(gate + cond * p.gate_ld + ch, k);
    if (gs != nullptr) g_raw.load(gs + cond * p.gate_shift_ld + ch, k);
  };
  auto fetch = [&] {
    const int k = left > 0 ? n : 0;
    const long long o = static_cast<long long>(row) * p.c + ch, e = static_cast<long long>(row) * groups + ch / kGroup8;
    if (dr != nullptr) dr_raw.load(dr + o, k);
    if (p.norm != kNoNorm) {
      dy_raw.load(dy + o, k);
      if (p.r_e != nullptr) r_raw.load8(static_cast<const uint8_t*>(p.r) + o, p.r_e + e, k);
      else r_raw.load(r + o, k);
    }
    if (p.dgate != nullptr) {
      if (p.u_e != nullptr) u_raw.load8(static_cast<const uint8_t*>(p.u) + o, p.u_e + e, k);
      else u_raw.load(u + o, k);
    }
    if (p.x != nullptr) {
      if (p.x_e != nullptr) x_raw.load8(static_cast<const uint8_t*>(p.x) + o, p.x_e + e, k);
      else x_raw.load(x + o, k);
    }
  };
  if (set < p.sets) {
    enter();
    fetch();
    if (OWN) gates();
  }
  int turn = 0;
  while (set < p.sets) {
    float t[N], v[N], d[N], z[N], slope_m[OWN ? N : 1], slope_u[OWN ? N : 1];
    const unsigned this_row = row, this_cond = cond;
    const int here = left > 0 ? n : 0, cond_here = there ? n : 0;
    const bool fresh = at == 0;
    if (fresh) {
      if (!OWN) gates();
      if (gate != nullptr) {
        gate_raw.values(t);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const Gate q = gate_at(t[i]);
          open[i] = q.open;
          if (OWN) slope_u[i] = q.slope;
        }
      }
      if (gs != nullptr) {
        g_raw.values(t);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const Gate q = gate_at(t[i]);
          m[i] = q.open;
          if (OWN) slope_m[i] = q.slope;
        }
      }
    }
    if (dr != nullptr) {
      dr_raw.values(t);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = 0.f;
    }
    float uv[N], xv[N];
    if (p.norm != kNoNorm) {
      dy_raw.values(d);
      if (p.r_e != nullptr) r_raw.values_of_8(z);
      else r_raw.values(z);
    }
    if (p.dgate != nullptr) {
      if (p.u_e != nullptr) u_raw.values_of_8(uv);
      else u_raw.values(uv);
    }
    if (p.x != nullptr) {
      if (p.x_e != nullptr) x_raw.values_of_8(xv);
      else x_raw.values(xv);
    }
    // on to the next row, whose loads have to stand before this one's stores
    bool last = OWN;
    if (OWN || ++at == p.chunk) {
      last = true;
      at = 0;
      set += step;
      if (set < p.sets) {
        enter();
        if (OWN) gates();
      }
    } else {
      --left;
      row += p.share.l;
    }
    if (set < p.sets) fetch();

    if (p.norm != kNoNorm) {
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[0] += z[i];
        s[1] = fmaf(d[i], m[i], s[1]);
      }
      team_sum<LANES>(s, room, group, turn);
      turn ^= 1;
      const float mean = s[0] * inv_c, mean_g = s[1] * inv_c;
      s[0] = s[1] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        z[i] = (VEC ? n > 0 : i < n) ? z[i] - mean : 0.f;
        s[0] = fmaf(z[i], z[i], s[0]);
        s[1] = fmaf(d[i] * m[i], z[i], s[1]);
      }
      team_sum<LANES>(s, room, group, turn);
      turn ^= 1;
      const float rstd = rsqrtf(fmaf(s[0], inv_c, p.eps)), mean_gz = s[1] * inv_c * rstd;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        z[i] *= rstd;
        t[i] = fmaf(rstd, fmaf(d[i], m[i], -mean_g) - z[i] * mean_gz, t[i]);
      }
      if (OWN && adaptive) {
        if (p.dgate_shift != nullptr) {
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = d[i] * z[i] * slope_m[i];
          TC* o = static_cast<TC*>(p.dgate_shift) + static_cast<long long>(this_row) * 2 * p.c + ch;
          store_piece<VEC>(o, v, here);
          store_piece<VEC>(o + p.c, d, here);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a0[i] = fmaf(d[i], here > 0 ? z[i] : 0.f, a0[i]);      // (z of no row is not a number where eps is zero)
          a1[i] += d[i];
        }
      }
    }
    const long long o = static_cast<long long>(this_row) * p.c + ch;
    if (p.dgate != nullptr) {
      if (OWN) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t[i] * uv[i] * slope_u[i];
        store_piece<VEC>(static_cast<TC*>(p.dgate) + o, v, here);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) a2[i] = fmaf(here > 0 ? t[i] : 0.f, uv[i], a2[i]);
      }
    }
    if (p.x != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) a3[i] = fmaf(here > 0 ? t[i] : 0.f, xv[i], a3[i]);
    }
    if (p.du != nullptr) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = t[i] * open[i];
      store_piece<VEC>(static_cast<TC*>(p.du) + o, v, here);
    }
    if (p.dx != nullptr) {
      if (p.scale != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] *= i < n ? p.scale[ch + i] : 0.f;
      }
      store_piece<VEC>(static_cast<TS*>(p.dx) + o, t, here);
    }
    if constexpr (!OWN) {
      if (last) {
        // the gates' gradients from the sums over their samples; the logits once more, for their slopes
        bool mine = true;
        if (p.split) {
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const float* a = k == 0 ? a0 : k == 1 ? a1 : a2;
            s_sum[k][threadIdx.x * 2] = make_float4(a[0], a[1], a[2], a[3]);
            s_sum[k][threadIdx.x * 2 + 1] = make_float4(a[4], a[5], a[6], a[7]);
          }
          __syncthreads();
          mine = group == 0;
          if (mine) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              if (k < 2 && !adaptive) continue;
              float* a = k == 0 ? a0 : k == 1 ? a1 : a2;
              for (int q = 1; q < T::kGroups; ++q) {
                const float4 lo = s_sum[k][(q * T::kGroupLanes + threadIdx.x) * 2], hi = s_sum[k][(q * T::kGroupLanes + threadIdx.x) * 2 + 1];
                a[0] += lo.x;
                a[1] += lo.y;
                a[2] += lo.z;
                a[3] += lo.w;
                a[4] += hi.x;
                a[5] += hi.y;
                a[6] += hi.z;
                a[7] += hi.w;
              }
            }
          }
          __syncthreads();
        }
        if (mine && adaptive && p.dgate_shift != nullptr) {
          g_raw.load(gs + this_cond * p.gate_shift_ld + ch, cond_here);
          g_raw.values(v);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = a0[i] * gate_at(v[i]).slope;
          TC* q = static_cast<TC*>(p.dgate_shift) + static_cast<long long>(this_cond) * 2 * p.c + ch;
          store_piece<VEC>(q, v, cond_here);
          store_piece<VEC>(q + p.c, a1, cond_here);
        }
        if (mine && p.dgate != nullptr) {
          gate_raw.load(gate + this_cond * p.gate_ld + ch, cond_here);
          gate_raw.values(v);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = a2[i] * gate_at(v[i]).slope;
          store_piece<VEC>(static_cast<TC*>(p.dgate) + static_cast<long long>(this_cond) * p.c + ch, v, cond_here);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a2[i] = 0.f;
          if (adaptive) a0[i] = a1[i] = 0.f;
        }
      }
    }
  }

  if (p.partial != nullptr) {
    // the block's teams in their order
    float* flat = reinterpret_cast<float*>(s_sum[0]);      // [team][LANES * 8]
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const float* a = k == 0 ? a0 : k == 1 ? a1 : a3;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) flat[(group * T::kTeams + team) * LANES * N + ch + i] = a[i];
      __syncthreads();
      for (int i = threadIdx.x; i < p.c; i += T::kThreads) {
        float s = 0.f;
#pragma unroll 4
        for (int q = 0; q < T::kGroups * T::kTeams; ++q) s += flat[q * LANES * N + i];
        p.partial[(static_cast<long long>(blockIdx.x) * 3 + k) * p.c + i] = s;
      }
    }
  }
}

// The three sums (any may have no place) from the blocks' rows of partial sums, in the order of the blocks.
__global__ void __launch_bounds__(1024) residual_norm_sum_kernel(const float* partial, float* d0, float* d1, float* d2, int blocks, int c) {
  __shared__ float s[32][33];
  grid_dependency_enter();
  const int col = blockIdx.x * 32 + threadIdx.x % 32, part = threadIdx.x / 32;
  float t = 0.f;
  if (col < 3 * c) {
#pragma unroll 4
    for (int b = part; b < blocks; b += 32) t += partial[static_cast<long long>(b) * 3 * c + col];
  }
  s[part][threadIdx.x % 32] = t;
  __syncthreads();
  if (part == 0 && col < 3 * c) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += s[k][threadIdx.x];
    float* d = col < c ? d0 : col < 2 * c ? d1 : d2;
    if (d != nullptr) d[col % c] = t;
  }
}

constexpr int kBlocksPerSm = 4;      // at most: the workspace's partial sums are sized by it
constexpr int kMostSms = 160;

struct Sums {
  float *dweight, *dbias, *dscale;
};

template <typename TS, typename TC, int LANES, bool VEC, bool OWN>
int launch(cudaStream_t stream, GradParams p, const Sums& sums) {
  using T = Teams<LANES>;
  auto kernel = residual_norm_grad_kernel<TS, TC, LANES, VEC, OWN>;
  static std::once_flag once;
  static int held = 1;
  std::call_once(once, [&] {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, T::kThreads, 0) != cudaSuccess) cudaGetLastError();
    held = held < 1 ? 1 : held > kBlocksPerSm ? kBlocksPerSm : held;
  });
  const unsigned most = static_cast<unsigned>(sm_count() < kMostSms ? sm_count() : kMostSms) * held;
  const unsigned rows = p.share.cond_rows, teams = T::kGroups * T::kTeams;
  p.split = p.share.samples > 1 && rows < most * teams;
  p.chunk = p.split ? cdiv(p.share.samples, T::kGroups) : p.share.samples;
  p.sets = (rows + T::kTeams - 1) / T::kTeams;
  const unsigned want = p.split ? p.sets : (p.sets + T::kGroups - 1) / T::kGroups, blocks = want < most ? want : most;
  {
    LaunchScope scope(stream, "residual_norm_grad");
    KFB_TRY(launch_kernel(stream, kernel, blocks, T::kThreads, 0, p));
  }
  if (p.partial != nullptr) {
    LaunchScope scope(stream, "residual_norm_sum");
    KFB_TRY(launch_kernel(stream, residual_norm_sum_kernel, cdiv(3 * p.c, 32), 1024, 0, const_cast<const float*>(p.partial), sums.dweight, sums.dbias,
                          sums.dscale, static_cast<int>(blocks), p.c));
  }
  return KFB_OK;
}

template <typename TS, typename TC, int LANES, bool VEC>
int launch_own(cudaStream_t stream, const GradParams& p, const Sums& sums) {
  return p.share.samples == 1 ? launch<TS, TC, LANES, VEC, true>(stream, p, sums) : launch<TS, TC, LANES, VEC, false>(stream, p, sums);
}

template <typename TS, typename TC>
int dispatch(cudaStream_t stream, const GradParams& p, const Sums& sums) {
  auto of = [](const void* q, const uint8_t* e) { return reinterpret_cast<uintptr_t>(q) << (e != nullptr ? 1 : 0); };   // bytes: 8-byte boundaries do
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.dr) | reinterpret_cast<uintptr_t>(p.dy) | of(p.r, p.r_e) | of(p.u, p.u_e) | of(p.x, p.x_e) |
                       reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.gate_shift) | reinterpret_cast<uintptr_t>(p.dx) |
                       reinterpret_cast<uintptr_t>(p.du) | reinterpret_cast<uintptr_t>(p.dgate) | reinterpret_cast<uintptr_t>(p.dgate_shift) |
                       static_cast<uintptr_t>((p.gate_ld | p.gate_shift_ld) * sizeof(TC));
  if (p.c % 8 == 0 && (at & 15) == 0) {
    if (p.c <= 64) return launch_own<TS, TC, 8, true>(stream, p, sums);
    if (p.c <= 128) return launch_own<TS, TC, 16, true>(stream, p, sums);
    if (p.c <= 256) return launch_own<TS, TC, 32, true>(stream, p, sums);
    if (p.c <= 512) return launch_own<TS, TC, 64, true>(stream, p, sums);
    if (p.c <= 768) return launch_own<TS, TC, 96, true>(stream, p, sums);
    return launch_own<TS, TC, 128, true>(stream, p, sums);
  }
  return p.c <= 256 ? launch_own<TS, TC, 32, false>(stream, p, sums) : launch_own<TS, TC, 128, false>(stream, p, sums);
}

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API size_t kfb_residual_norm_bwd_workspace_bytes(int c) {
  return align_up(static_cast<size_t>(kMostSms) * kBlocksPerSm * 3 * (c > 0 ? c : 0) * sizeof(float), 256);
}

KFB_API int kfb_residual_norm_bwd(const void* dr, const void* dy, const void* r, const void* r_exponents, const void* u, const void* u_exponents,
                                  const void* x, const void* x_exponents, const void* gate, long long gate_ld, const float* scale,
                                  const float* weight, const void* gate_shift, long long gate_shift_ld, void* dx, void* du, void* dgate,
                                  void* dgate_shift, float* dweight, float* dbias, float* dscale, void* workspace, size_t workspace_bytes,
                                  long long rows, int c, int samples, int l, float eps, int norm, int stream_dtype, int compute_dtype, void* stream) {
  KFB_CHECK_ARG(rows >= 0 && rows < (1ll << 31) && c > 0 && samples > 0 && l > 0 && rows % (static_cast<long long>(samples) * l) == 0,
                "residual_norm_bwd: rows %lld of %d channels, %d samples of %d tokens", rows, c, samples, l);
  if (c > 1024) {
    set_error("residual_norm_bwd: channel count %d above 1024 is not supported", c);
    return KFB_ERR_UNSUPPORTED;
  }
  KFB_CHECK_ARG((stream_dtype == KFB_BF16 && compute_dtype == KFB_BF16) || (stream_dtype == KFB_FP32 && (compute_dtype == KFB_BF16 || compute_dtype == KFB_FP32)),
                "residual_norm_bwd: dtypes %d and %d", stream_dtype, compute_dtype);
  KFB_CHECK_ARG(norm >= kNoNorm && norm <= kAdaptiveNorm && (norm == kAdaptiveNorm) == (gate_shift != nullptr) &&
                    (norm == kAffineNorm || (weight == nullptr && dweight == nullptr && dbias == nullptr)) && (norm == kAdaptiveNorm || dgate_shift == nullptr),
                "residual_norm_bwd: norm %d with other parameters", norm);
  KFB_CHECK_ARG((gate == nullptr || gate_ld >= c) && (gate_shift == nullptr || gate_shift_ld >= 2ll * c), "residual_norm_bwd: gate rows %lld and %lld apart",
                gate_ld, gate_shift_ld);
  const bool sums = dweight != nullptr || dbias != nullptr || dscale != nullptr;
  const bool shared = samples > 1 && (gate != nullptr || gate_shift != nullptr);
  cudaStream_t s = as_stream(stream);
  if (rows == 0) {
    for (float* d : {dweight, dbias, dscale})
      if (d != nullptr) KFB_CUDA(cudaMemsetAsync(d, 0, static_cast<size_t>(c) * 4, s));
    return KFB_OK;
  }
  KFB_CHECK_ARG((norm == kNoNorm || (dy != nullptr && r != nullptr)) && (norm != kNoNorm || dr != nullptr), "residual_norm_bwd: null tensor");
  KFB_CHECK_ARG(dgate == nullptr || (gate != nullptr && u != nullptr), "residual_norm_bwd: a gate's gradient needs the gate and what it multiplies");
  KFB_CHECK_ARG(dscale == nullptr || x != nullptr, "residual_norm_bwd: the scale's gradient needs x");
  KFB_CHECK_ARG(!sums || (workspace != nullptr && workspace_bytes >= kfb_residual_norm_bwd_workspace_bytes(c)), "residual_norm_bwd: workspace %zu < %zu bytes",
                workspace_bytes, kfb_residual_norm_bwd_workspace_bytes(c));
  KFB_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "residual_norm_bwd: workspace must be 256-byte aligned");
  GradParams p = {};
  p.dr = dr;
  p.dy = norm != kNoNorm ? dy : nullptr;
  p.r = norm != kNoNorm ? r : nullptr;
  p.r_e = norm != kNoNorm ? static_cast<const uint8_t*>(r_exponents) : nullptr;
  p.u = dgate != nullptr ? u : nullptr;
  p.u_e = dgate != nullptr ? static_cast<const uint8_t*>(u_exponents) : nullptr;
  p.x = dscale != nullptr ? x : nullptr;
  p.x_e = dscale != nullptr ? static_cast<const uint8_t*>(x_exponents) : nullptr;
  p.gate = gate;
  p.gate_shift = gate_shift;
  p.scale = scale;
  p.weight = weight;
  p.gate_ld = gate != nullptr ? gate_ld : 0;
  p.gate_shift_ld = gate_shift != nullptr ? gate_shift_ld : 0;
  p.dx = dx;
  p.du = du;
  p.dgate = dgate;
  p.dgate_shift = dgate_shift;
  p.partial = sums ? static_cast<float*>(workspace) : nullptr;
  p.share = {static_cast<unsigned>(shared ? rows / samples : rows), static_cast<unsigned>(l), shared ? samples : 1};
  p.c = c;
  p.norm = norm;
  p.eps = eps;
  const Sums to = {dweight, dbias, dscale};
  if (stream_dtype == KFB_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(s, p, to);
  return compute_dtype == KFB_BF16 ? dispatch<float, __nv_bfloat16>(s, p, to) : dispatch<float, float>(s, p, to);
}

}  // extern "C"
