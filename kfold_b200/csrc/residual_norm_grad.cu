// The gradient of residual_norm.cu.  With z = (r - mean) rstd of the stored r, m the factor of the norm and s = sigmoid(gate):
//   g = m dy,  t = dr + rstd (g - mean(g) - z mean(g z)),  dx = scale t,  du = s t,
//   dgate = s (1 - s) sum(t u),  d gate_shift = [m (1 - m) sum(dy z) | sum(dy)]  over the samples that share the row,
//   dweight = sum(dy z),  dbias = sum(dy),  dscale = sum(t x)  over all rows.
//
// What bounds it: dr, dy, r and u in, dx and du out, HBM.  Row statistics come from r again.  r, u and x may be the tensors or rows kept in 8 bits
// (row_teams.cuh), which are taken apart in registers.
// Split: residual_norm.cuh says how rows are walked and come in.  A team keeps the sums over the samples of a gate row in registers; where these samples are
// cut into pieces, a piece leaves its sums in the workspace and a second kernel adds them in the pieces' order.  Sums over all rows stay in registers from row
// to row; a block leaves a row of partial sums, added up likewise.  No atomics: the order hangs on the sizes alone.
#include <mutex>

#include "ops_common.cuh"
#include "residual_norm.cuh"

namespace kfb {
namespace {

struct GradParams {
  const void *dr, *dy, *r, *u, *x, *gate, *gate_shift;
  const uint8_t *r_e, *u_e, *x_e;      // exponents of those that are kept in 8 bits
  const float *scale, *weight;
  long long gate_ld, gate_shift_ld;
  void *dx, *du, *dgate, *dgate_shift;
  float* partial;                      // [block][3][c]: sums of dy z, dy, t x
  float* pieces;                       // [unit][3][c]: a piece's sums of dy z, dy, t u; null: a gate row's samples are one piece
  RowPlan plan;
  int c, norm;
  float eps;
  int slots, s_dy, s_r, s_u, s_x, s_gate, s_g;    // slots of a stage, and the first of each tensor (dr: 0)
  int words;                           // exponents come in words of four (a row's are whole words, and start on one)
};

// OWN: a row has gates of its own.
template <typename TS, typename TC, int LANES, bool VEC, bool OWN>
__global__ void __launch_bounds__(Teams<LANES>::kThreads, 2) residual_norm_grad_kernel(const GradParams p) {
  using T = Teams<LANES>;
  constexpr int N = kPiece, kThreads = T::kThreads, kDepth = OWN ? 3 : 4;      // rows on their way for a team, the one in work among them
  __shared__ float room[2][T::kGroups][T::kWarps][2];
  extern __shared__ uint4 ring_memory[];
  grid_dependency_enter();
  const int group = threadIdx.x / T::kGroupLanes, sub = threadIdx.x % LANES, team = threadIdx.x % T::kGroupLanes / LANES;
  const int ch = sub * N, n = min(max(p.c - ch, 0), N), groups = groups8(p.c), e_shift = ch / kGroup8 % 4 * 8;
  const float inv_c = 1.0f / static_cast<float>(p.c);
  const TS* dr = static_cast<const TS*>(p.dr);
  const TC *dy = static_cast<const TC*>(p.dy), *gate = static_cast<const TC*>(p.gate), *gs = static_cast<const TC*>(p.gate_shift);
  const bool adaptive = p.norm == kAdaptiveNorm;
  uint4* ring = ring_memory + threadIdx.x;

  float m[N], open[OWN ? 1 : N], a0[N], a1[N], a2[OWN ? 1 : N], a3[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = p.weight != nullptr && i < n ? p.weight[ch + i] : 1.f;
    a0[i] = a1[i] = a3[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < (OWN ? 1 : N); ++i) {
    open[i] = 1.f;
    a2[i] = 0.f;
  }

  const unsigned step = gridDim.x * T::kGroups;
  Walk<LANES, OWN> here, ahead;
  here.set = blockIdx.x * T::kGroups + group;
  if (here.set < p.plan.sets) here.enter(p.plan, team);
  ahead = here;
  // a tensor of the stream's or the blocks' type, or its rows in 8 bits, into its slots and out of them
  auto copy = [&](auto tag, int slot, int stage, const void* q, const uint8_t* e, unsigned row, bool there) {
    using E = decltype(tag);
    uint4* to = ring + (stage * p.slots + slot) * kThreads;
    const long long o = static_cast<long long>(row) * p.c + ch;
    if (e == nullptr) {
      ring_copy<E, VEC>(to, kThreads, static_cast<const E*>(q) + o, there);
    } else {
      copy_async<8>(to, static_cast<const uint8_t*>(q) + o, there);
      if (p.words) copy_async<4>(reinterpret_cast<uint32_t*>(to) + 2, e + static_cast<long long>(row) * groups + (ch / kGroup8 & ~3), there);
    }
  };
  auto take = [&](auto tag, int slot, int stage, const void* q, const uint8_t* e, float* v) {
    using E = decltype(tag);
    Piece<E, VEC> raw;
    const int k = here.left > 0 ? n : 0;
    [[maybe_unused]] const uint4* from = ring + (stage * p.slots + slot) * kThreads;
    [[maybe_unused]] const long long o = static_cast<long long>(here.row) * p.c + ch;
    const uint8_t* ep = e == nullptr ? nullptr : e + static_cast<long long>(here.row) * groups + ch / kGroup8;
    if (e == nullptr) {
      if constexpr (VEC) raw.take(from, kThreads);
      else raw.load(static_cast<const E*>(q) + o, k);
      raw.values(v);
    } else {
      if constexpr (VEC) {
        raw.take8(from, e_shift);
        if (!p.words) raw.w[2] = k > 0 ? *ep : 0u;
      } else {
        raw.load8(static_cast<const uint8_t*>(q) + o, ep, k);
      }
      raw.values_of_8(v);
    }
  };
  auto fetch = [&](int stage) {
    if (ahead.set < p.plan.sets) {
      const bool there = ahead.left > 0 && n > 0;
      if (dr != nullptr) copy(TS{}, 0, stage, dr, nullptr, ahead.row, there);
      if (p.norm != kNoNorm) {
        copy(TC{}, p.s_dy, stage, dy, nullptr, ahead.row, there);
        copy(TS{}, p.s_r, stage, p.r, p.r_e, ahead.row, there);
      }
      if (p.dgate != nullptr) copy(TC{}, p.s_u, stage, p.u, p.u_e, ahead.row, there);
      if (p.x != nullptr) copy(TS{}, p.s_x, stage, p.x, p.x_e, ahead.row, there);
      if (OWN) {
        if (gate != nullptr) ring_copy<TC, VEC>(ring + (stage * p.slots + p.s_gate) * kThreads, kThreads, gate + ahead.row * p.gate_ld + ch, there);
        if (gs != nullptr) ring_copy<TC, VEC>(ring + (stage * p.slots + p.s_g) * kThreads, kThreads, gs + ahead.row * p.gate_shift_ld + ch, there);
      }
      ahead.next(p.plan, team, step);
    }
    copy_async_done();
  };
  // logits of this row's gate, or of the norm's
  auto logits = [&](const TC* table, long long ld, int slot, int stage, unsigned gate_row, int k, float* v) {
    Piece<TC, VEC> raw;
    if (OWN && VEC) raw.take(ring + (stage * p.slots + slot) * kThreads, kThreads);
    else raw.load(table + gate_row * ld + ch, k);
    raw.values(v);
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
    }
    const int k = here.left > 0 ? n : 0;
    const bool row_there = here.left > 0;
    const long long o = static_cast<long long>(here.row) * p.c + ch;
    float t[N], v[N];
    if (!OWN && here.at == 0) {
      const unsigned gate_row = here.gate_row(p.plan);
      if (gate != nullptr) {
        logits(gate, p.gate_ld, 0, 0, gate_row, k, t);
#pragma unroll
        for (int i = 0; i < (OWN ? 1 : N); ++i) open[i] = gate_at(t[i]).open;
      }
      if (gs != nullptr) {
        logits(gs, p.gate_shift_ld, 0, 0, gate_row, k, t);
#pragma unroll
        for (int i = 0; i < N; ++i) m[i] = gate_at(t[i]).open;
      }
    }
    if (OWN && gs != nullptr) {
      logits(gs, p.gate_shift_ld, p.s_g, stage, here.row, k, t);
#pragma unroll
      for (int i = 0; i < N; ++i) m[i] = gate_at(t[i]).open;
    }
    if (dr != nullptr) {
      take(TS{}, 0, stage, dr, nullptr, t);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) t[i] = 0.f;
    }
    if (p.norm != kNoNorm) {
      float d[N], z[N];
      take(TC{}, p.s_dy, stage, dy, nullptr, d);
      take(TS{}, p.s_r, stage, p.r, p.r_e, z);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[0] += z[i];
        s[1] = fmaf(d[i], m[i], s[1]);
      }
      team_sum<LANES>(s, room, group, 0);
      const float mean = s[0] * inv_c, mean_g = s[1] * inv_c;
      s[0] = s[1] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        z[i] = (VEC ? n > 0 : i < n) ? z[i] - mean : 0.f;
        s[0] = fmaf(z[i], z[i], s[0]);
        s[1] = fmaf(d[i] * m[i], z[i], s[1]);
      }
      team_sum<LANES>(s, room, group, 1);
      const float rstd = rsqrtf(fmaf(s[0], inv_c, p.eps)), mean_gz = s[1] * inv_c * rstd;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        z[i] *= rstd;
        t[i] = fmaf(rstd, fmaf(d[i], m[i], -mean_g) - z[i] * mean_gz, t[i]);
      }
      if (OWN && adaptive) {
        if (p.dgate_shift != nullptr) {
          logits(gs, p.gate_shift_ld, p.s_g, stage, here.row, k, v);
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = d[i] * z[i] * gate_at(v[i]).slope;
          TC* q = static_cast<TC*>(p.dgate_shift) + static_cast<long long>(here.row) * 2 * p.c + ch;
          store_piece<VEC>(q, v, k);
          store_piece<VEC>(q + p.c, d, k);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a0[i] = fmaf(d[i], row_there ? z[i] : 0.f, a0[i]);      // (z of no row is not a number where eps is zero)
          a1[i] += d[i];
        }
      }
    }
    if (p.dgate != nullptr) {
      take(TC{}, p.s_u, stage, p.u, p.u_e, v);
      if constexpr (OWN) {
        float s[N];
        logits(gate, p.gate_ld, p.s_gate, stage, here.row, k, s);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t[i] * v[i] * gate_at(s[i]).slope;
        store_piece<VEC>(static_cast<TC*>(p.dgate) + o, v, k);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) a2[i] = fmaf(row_there ? t[i] : 0.f, v[i], a2[i]);
      }
    }
    if (p.x != nullptr) {
      take(TS{}, p.s_x, stage, p.x, p.x_e, v);
#pragma unroll
      for (int i = 0; i < N; ++i) a3[i] = fmaf(row_there ? t[i] : 0.f, v[i], a3[i]);
    }
    if (p.du != nullptr) {
      if (OWN && gate != nullptr) {
        logits(gate, p.gate_ld, p.s_gate, stage, here.row, k, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t[i] * gate_at(v[i]).open;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t[i] * open[OWN ? 0 : i];
      }
      store_piece<VEC>(static_cast<TC*>(p.du) + o, v, k);
    }
    if (p.dx != nullptr) {
      if (p.scale != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] *= i < n ? p.scale[ch + i] : 0.f;
      }
      store_piece<VEC>(static_cast<TS*>(p.dx) + o, t, k);
    }
    if constexpr (!OWN) {
      if (here.at + 1 == p.plan.chunk) {
        // the end of a piece: the gates' gradients from the sums over their samples, the logits once more for their slopes; or the sums for the second kernel
        const bool there = here.unit < p.plan.units;
        const int kk = there ? n : 0;
        const unsigned gate_row = here.gate_row(p.plan);
        if (p.pieces != nullptr) {
          float* q = p.pieces + static_cast<long long>(there ? here.unit : 0) * 3 * p.c + ch;
          if (adaptive) {
            store_piece<VEC>(q, a0, kk);
            store_piece<VEC>(q + p.c, a1, kk);
          }
          if (p.dgate != nullptr) store_piece<VEC>(q + 2 * p.c, a2, kk);
        } else {
          if (adaptive && p.dgate_shift != nullptr) {
            logits(gs, p.gate_shift_ld, 0, 0, gate_row, kk, v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = a0[i] * gate_at(v[i]).slope;
            TC* q = static_cast<TC*>(p.dgate_shift) + static_cast<long long>(gate_row) * 2 * p.c + ch;
            store_piece<VEC>(q, v, kk);
            store_piece<VEC>(q + p.c, a1, kk);
          }
          if (p.dgate != nullptr) {
            logits(gate, p.gate_ld, 0, 0, gate_row, kk, v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = a2[i] * gate_at(v[i]).slope;
            store_piece<VEC>(static_cast<TC*>(p.dgate) + static_cast<long long>(gate_row) * p.c + ch, v, kk);
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a2[i] = 0.f;
          if (adaptive) a0[i] = a1[i] = 0.f;
        }
      }
    }
    here.next(p.plan, team, step);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
  }

  if (p.partial != nullptr) {
    // the block's teams in their order; the ring's memory, in which nothing is on its way any more
    copy_async_wait<0>();
    float* flat = reinterpret_cast<float*>(ring_memory);      // [team][LANES * 8]
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const float* a = j == 0 ? a0 : j == 1 ? a1 : a3;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) flat[(group * T::kTeams + team) * LANES * N + ch + i] = a[i];
      __syncthreads();
      for (int i = threadIdx.x; i < p.c; i += kThreads) {
        float s = 0.f;
#pragma unroll 4
        for (int q = 0; q < T::kGroups * T::kTeams; ++q) s += flat[q * LANES * N + i];
        p.partial[(static_cast<long long>(blockIdx.x) * 3 + j) * p.c + i] = s;
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

// The gates' gradients of rows whose samples were cut into pieces, in the order of the pieces.  A thread takes a channel of a row.
template <typename TC>
__global__ void __launch_bounds__(256) residual_norm_gates_kernel(const float* pieces, const TC* gate, long long gate_ld, const TC* gs, long long gs_ld, TC* dgate,
                                                                  TC* dgs, unsigned gate_rows, int chunks, int c) {
  grid_dependency_enter();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < static_cast<long long>(gate_rows) * c; i += gridDim.x * 256ll) {
    const unsigned row = static_cast<unsigned>(i / c);
    const int ch = static_cast<int>(i - static_cast<long long>(row) * c);
    float s[3] = {0.f, 0.f, 0.f};
    const float* q = pieces + static_cast<long long>(row) * chunks * 3 * c + ch;
#pragma unroll 4
    for (int k = 0; k < chunks; ++k, q += 3ll * c) {
      if (dgs != nullptr) {
        s[0] += q[0];
        s[1] += q[c];
      }
      if (dgate != nullptr) s[2] += q[2 * c];
    }
    float v;
    if (dgs != nullptr) {
      TC* d = dgs + static_cast<long long>(row) * 2 * c + ch;
      v = s[0] * gate_at(static_cast<float>(gs[row * gs_ld + ch])).slope;
      store_vec<1>(d, &v);
      store_vec<1>(d + c, &s[1]);
    }
    if (dgate != nullptr) {
      v = s[2] * gate_at(static_cast<float>(gate[row * gate_ld + ch])).slope;
      store_vec<1>(dgate + static_cast<long long>(row) * c + ch, &v);
    }
  }
}

constexpr int kBlocksPerSm = 4;      // at most: the workspace's partial sums are sized by it
constexpr int kMostSms = 160;
constexpr int kMostRing = 216 * 1024;
// Pieces of gate rows' samples, at most: two for each team that is at work (row_plan), of which a block has so many.
constexpr long long most_units(int c) { return 2ll * kMostSms * kBlocksPerSm * (c <= 64 ? 32 : c <= 128 ? 16 : c <= 256 ? 8 : c <= 512 ? 4 : c <= 768 ? 3 : 2); }

struct Sums {
  float *dweight, *dbias, *dscale;
};

template <typename TS, typename TC, int LANES, bool VEC, bool OWN>
int launch(cudaStream_t stream, GradParams p, const Sums& sums, long long rows, int samples, int l) {
  using T = Teams<LANES>;
  constexpr auto kernel = residual_norm_grad_kernel<TS, TC, LANES, VEC, OWN>;
  constexpr int kS = sizeof(TS) / 2, kC = sizeof(TC) / 2, kDepth = OWN ? 3 : 4, kFlat = T::kThreads * kPiece * 4;
  static std::once_flag once;
  static int held = 1;
  std::call_once(once, [&] {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, T::kThreads, 0) != cudaSuccess) cudaGetLastError();
    held = held < 1 ? 1 : held > kBlocksPerSm ? kBlocksPerSm : held;
  });
  // (a row in 8 bits takes one slot)
  int slots = p.dr != nullptr ? kS : 0;
  auto place = [&](bool there, bool small, int size) {
    const int at = slots;
    slots += !there ? 0 : small ? 1 : size;
    return at;
  };
  p.s_dy = place(p.norm != kNoNorm, false, kC);
  p.s_r = place(p.norm != kNoNorm, p.r_e != nullptr, kS);
  p.s_u = place(p.dgate != nullptr, p.u_e != nullptr, kC);
  p.s_x = place(p.x != nullptr, p.x_e != nullptr, kS);
  p.s_gate = place(OWN && p.gate != nullptr, false, kC);
  p.s_g = place(OWN && p.gate_shift != nullptr, false, kC);
  p.slots = slots;
  int smem = VEC ? kDepth * slots * T::kThreads * 16 : 0;
  if (p.partial != nullptr && smem < kFlat) smem = kFlat;
  KFB_TRY(allow_smem<kernel>(kMostRing));
  const int fit = smem > 0 ? kMostRing / smem : held, blocks_per_sm = held < fit ? held : fit < 1 ? 1 : fit;
  const long long most = static_cast<long long>(sm_count() < kMostSms ? sm_count() : kMostSms) * blocks_per_sm, teams = T::kGroups * T::kTeams;
  p.plan = row_plan(rows, samples, l, most * teams, T::kTeams);
  const bool gates = p.dgate != nullptr || p.dgate_shift != nullptr;
  if (p.plan.chunks == 1 || !gates) p.pieces = nullptr;
  else KFB_CHECK_ARG(p.plan.units <= most_units(p.c), "residual_norm_bwd: %u pieces", p.plan.units);
  const long long want = (p.plan.sets + T::kGroups - 1) / T::kGroups;
  const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
  {
    LaunchScope scope(stream, "residual_norm_grad");
    KFB_TRY(launch_kernel(stream, kernel, blocks, T::kThreads, smem, p));
  }
  if (p.pieces != nullptr) {
    const long long n = (static_cast<long long>(p.plan.gate_rows) * p.c + 255) / 256, grid = 4ll * sm_count();
    LaunchScope scope(stream, "residual_norm_gates");
    KFB_TRY(launch_kernel(stream, residual_norm_gates_kernel<TC>, static_cast<unsigned>(n < grid ? n : grid), 256, 0, const_cast<const float*>(p.pieces),
                          static_cast<const TC*>(p.gate), p.gate_ld, static_cast<const TC*>(p.gate_shift), p.gate_shift_ld, static_cast<TC*>(p.dgate),
                          static_cast<TC*>(p.dgate_shift), p.plan.gate_rows, p.plan.chunks, p.c));
  }
  if (p.partial != nullptr) {
    LaunchScope scope(stream, "residual_norm_sum");
    KFB_TRY(launch_kernel(stream, residual_norm_sum_kernel, cdiv(3 * p.c, 32), 1024, 0, const_cast<const float*>(p.partial), sums.dweight, sums.dbias,
                          sums.dscale, static_cast<int>(blocks), p.c));
  }
  return KFB_OK;
}

template <typename TS, typename TC, int LANES, bool VEC>
int launch_own(cudaStream_t stream, const GradParams& p, const Sums& sums, long long rows, int samples, int l) {
  return samples == 1 ? launch<TS, TC, LANES, VEC, true>(stream, p, sums, rows, samples, l) : launch<TS, TC, LANES, VEC, false>(stream, p, sums, rows, samples, l);
}

template <typename TS, typename TC>
int dispatch(cudaStream_t stream, GradParams p, const Sums& sums, long long rows, int samples, int l) {
  auto of = [](const void* q, const uint8_t* e) { return reinterpret_cast<uintptr_t>(q) << (e != nullptr ? 1 : 0); };   // bytes: 8-byte boundaries do
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.dr) | reinterpret_cast<uintptr_t>(p.dy) | of(p.r, p.r_e) | of(p.u, p.u_e) | of(p.x, p.x_e) |
                       reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.gate_shift) | reinterpret_cast<uintptr_t>(p.dx) |
                       reinterpret_cast<uintptr_t>(p.du) | reinterpret_cast<uintptr_t>(p.dgate) | reinterpret_cast<uintptr_t>(p.dgate_shift) |
                       static_cast<uintptr_t>((p.gate_ld | p.gate_shift_ld) * sizeof(TC));
  p.words = groups8(p.c) % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.r_e) | reinterpret_cast<uintptr_t>(p.u_e) | reinterpret_cast<uintptr_t>(p.x_e)) & 3) == 0;
  if (p.c % 8 == 0 && (at & 15) == 0) {
    if (p.c <= 64) return launch_own<TS, TC, 8, true>(stream, p, sums, rows, samples, l);
    if (p.c <= 128) return launch_own<TS, TC, 16, true>(stream, p, sums, rows, samples, l);
    if (p.c <= 256) return launch_own<TS, TC, 32, true>(stream, p, sums, rows, samples, l);
    if (p.c <= 512) return launch_own<TS, TC, 64, true>(stream, p, sums, rows, samples, l);
    if (p.c <= 768) return launch_own<TS, TC, 96, true>(stream, p, sums, rows, samples, l);
    return launch_own<TS, TC, 128, true>(stream, p, sums, rows, samples, l);
  }
  return p.c <= 256 ? launch_own<TS, TC, 32, false>(stream, p, sums, rows, samples, l) : launch_own<TS, TC, 128, false>(stream, p, sums, rows, samples, l);
}

size_t partial_bytes(int c) { return align_up(static_cast<size_t>(kMostSms) * kBlocksPerSm * 3 * c * sizeof(float), 256); }

}  // namespace
}  // namespace kfb

using namespace kfb;

extern "C" {

KFB_API size_t kfb_residual_norm_bwd_workspace_bytes(long long rows, int c, int samples, int sums, int gates) {
  if (rows <= 0 || c <= 0 || c > 1024 || samples <= 0) return 0;
  const long long units = rows < most_units(c) ? rows : most_units(c);
  return (sums ? partial_bytes(c) : 0) + (gates && samples > 1 ? align_up(static_cast<size_t>(units) * 3 * c * sizeof(float), 256) : 0);
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
  const bool gates = shared && (dgate != nullptr || dgate_shift != nullptr);
  const size_t need = kfb_residual_norm_bwd_workspace_bytes(rows, c, samples, sums, gates);
  KFB_CHECK_ARG(need == 0 || (workspace != nullptr && workspace_bytes >= need), "residual_norm_bwd: workspace %zu < %zu bytes", workspace_bytes, need);
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
  p.pieces = gates ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (sums ? partial_bytes(c) : 0)) : nullptr;
  const int each = shared ? samples : 1;
  p.c = c;
  p.norm = norm;
  p.eps = eps;
  const Sums to = {dweight, dbias, dscale};
  if (stream_dtype == KFB_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(s, p, to, rows, each, l);
  return compute_dtype == KFB_BF16 ? dispatch<float, __nv_bfloat16>(s, p, to, rows, each, l) : dispatch<float, float>(s, p, to, rows, each, l);
}

}  // extern "C"
