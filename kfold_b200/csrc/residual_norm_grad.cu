// The gradient of residual_norm.cu.  With z = (r - mean) rstd of the stored r, m the factor of the norm and s = sigmoid(gate):
//   g = m dy,  t = dr + rstd (g - mean(g) - z mean(g z)),  dx = scale t,  du = s t,
//   dgate = s (1 - s) sum(t u),  d gate_shift = [m (1 - m) sum(dy z) | sum(dy)]  over the samples that share the row,
//   dweight = sum(dy z),  dbias = sum(dy),  dscale = sum(t x)  over all rows.
//
// What bounds it: dr, dy, r and u in, dx and du out, HBM.  Row statistics come from r again.  r, u and x may be the tensors or rows kept in 8 bits
// (row_teams.cuh), which are taken apart in registers.
// Split: residual_norm.cuh says how rows are walked and come in.  A team keeps the sums over the samples of a gate row in registers; where these samples are
// cut into pieces, a piece leaves its sums in the workspace and a second kernel adds them in the pieces' order.  Sums over all rows stay in registers from row
// to row; a block leaves a row of partial sums, added up likewise.  No atomics: the order hangs on the sizes alone.  The rows of residual_norm.cu, r from 8 bits where it was kept so:
//   shared gates   40 us, 3.9 TB/s: 254 registers, the sums of a gate row among them, leave eight warps an SM, whose sums over a row wait on one another
//   gates of their own, float32 stream   79 us, 5.0 TB/s          128 channels   31 us, 4.3 TB/s, of which 4 are the sums over the blocks
//   768 float32 channels, gates of their own   148 us, 4.6 TB/s                   shared   101 us, 3.4 TB/s
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
  int slots, s_dy, s_r, s_u, s_x, s_gate, s_g;    // slots of a stage, and the first of each tensor (dr: 0; s_x below zero: x is read as it lies)
  int s_scale;                         // behind the ring: this thread's sums of t x
  int words;                           // exponents come in words of four (a row's are whole words, and start on one)
};

template <typename TS, typename TC, int P, bool OWN>
constexpr int depth() { return ring_depth(P * 8 * (2 * sizeof(TS) + (OWN ? 4 : 2) * sizeof(TC)), OWN ? 3 : 2); }

template <typename TS, typename TC, int LANES, int P, bool VEC, int GATES>
__global__ void __launch_bounds__(kRowThreads, P == 1 ? 4 : P == 2 || (P == 3 && GATES == kOwnAdaptive) ? 3 : 2) residual_norm_grad_kernel(const GradParams p) {
  constexpr bool OWN = GATES != kSharedGates, kSums = GATES != kOwnAdaptive;      // (sums from row to row)
  constexpr int kDepth = depth<TS, TC, P, OWN>(), kC = sizeof(TC) / 2;
  constexpr int kStep = LANES * kPiece;      // channels from a lane's piece to its next
  extern __shared__ uint4 ring_memory[];
  grid_dependency_enter();
  const int warp = threadIdx.x / 32, ch = threadIdx.x % LANES * (VEC ? kPiece : 1), team = threadIdx.x % 32 / LANES, groups = groups8(p.c);
  const float inv_c = 1.0f / static_cast<float>(p.c);
  const TC *gate = static_cast<const TC*>(p.gate) + ch, *gs = static_cast<const TC*>(p.gate_shift) + ch;
  const bool gated = p.gate != nullptr, adaptive = GATES == kOwnAdaptive || (GATES == kSharedGates && p.norm == kAdaptiveNorm);
  const uint4* ring = ring_memory + threadIdx.x;
  const uint32_t ring_at = ptx::smem_u32(ring);
  float* scale_sums = reinterpret_cast<float*>(ring_memory + p.s_scale * kRowThreads) + threadIdx.x;      // [P * 8][thread]
  int inside[P];                             // channels of a piece
#pragma unroll
  for (int q = 0; q < P; ++q) inside[q] = channels_of<VEC>(p.c, ch + q * kStep);
  auto vector = [&](const float* v, int q, float other) {
    float f[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) f[i] = v != nullptr && i < inside[q] ? v[ch + q * kStep + i * channel_step<VEC>()] : other;
    return of_floats(f);
  };

  // m: what dy is multiplied by, weights or open gates; open: the output gates
  Pairs m[P], open[OWN ? 1 : P], a0[kSums ? P : 1], a1[kSums ? P : 1], a2[OWN ? 1 : P];
#pragma unroll
  for (int q = 0; q < P; ++q) {
    m[q] = vector(p.weight, q, 1.f);
    if (kSums) a0[kSums ? q : 0] = a1[kSums ? q : 0] = both(0.f);
    if (!OWN) open[OWN ? 0 : q] = both(1.f), a2[OWN ? 0 : q] = both(0.f);
    if (p.x != nullptr) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) scale_sums[(q * kPiece + i) * kRowThreads] = 0.f;
    }
  }

  const unsigned step = gridDim.x * (kRowThreads / 32);
  Walk<LANES, OWN> here, ahead;
  here.set = blockIdx.x * (kRowThreads / 32) + warp;
  if (here.set < p.plan.sets) here.enter(p.plan, team);
  ahead = here;
  auto fetch = [&](int stage) {
    if (ahead.set < p.plan.sets) {
      const uint32_t s = ring_at + stage * p.slots * kRowThreads * 16;
      const long long o = static_cast<long long>(ahead.row) * p.c + ch, e = static_cast<long long>(ahead.row) * groups;
      bool there[P];
#pragma unroll
      for (int q = 0; q < P; ++q) there[q] = ahead.left > 0 && inside[q] > 0;
      auto copy = [&](auto tag, int slot, const void* t, const uint8_t* exponents) {
        using E = decltype(tag);
        const uint32_t to = s + slot * kRowThreads * 16;
        if (exponents == nullptr) ring_copy<E, P, kStep>(to, static_cast<const E*>(t) + o, there);
        else ring_copy8<P, kStep>(to, static_cast<const uint8_t*>(t) + o, exponents + e, ch, p.words, there);
      };
      if (p.dr != nullptr) copy(TS{}, 0, p.dr, nullptr);
      if (p.norm != kNoNorm) {
        copy(TC{}, p.s_dy, p.dy, nullptr);
        copy(TS{}, p.s_r, p.r, p.r_e);
      }
      if (p.dgate != nullptr) copy(TC{}, p.s_u, p.u, p.u_e);
      if (p.x != nullptr && p.s_x >= 0) copy(TS{}, p.s_x, p.x, p.x_e);
      if (OWN && gated) ring_copy<TC, P, kStep>(s + p.s_gate * kRowThreads * 16, gate + ahead.row * p.gate_ld, there);
      if (OWN && adaptive) ring_copy<TC, P, kStep>(s + p.s_g * kRowThreads * 16, gs + ahead.row * p.gate_shift_ld, there);
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
    const bool row_there = here.left > 0;
    uint32_t r_ex[P];                        // r's exponents where they come in no words: asked for before the wait; nothing without a norm
    if constexpr (VEC) {
      fetch(stage == 0 ? kDepth - 1 : stage - 1);
      if (p.r_e != nullptr && !p.words) {
#pragma unroll
        for (int q = 0; q < P; ++q)
          r_ex[q] = row_there && inside[q] > 0 ? p.r_e[static_cast<long long>(here.row) * groups + (ch + q * kStep) / kGroup8] : 0u;
      }
      copy_async_wait<kDepth - 1>();
    } else {
      ahead.next(p.plan, team, step);
      if (ahead.set < p.plan.sets && ahead.left > 0) {
        const int lane = threadIdx.x % 32;
        const long long o = static_cast<long long>(ahead.row) * p.c;
        if (p.dr != nullptr) prefetch_row(static_cast<const TS*>(p.dr) + o, p.c, lane);
        if (p.norm != kNoNorm) {
          prefetch_row(static_cast<const TC*>(p.dy) + o, p.c, lane);
          if (p.r_e != nullptr) prefetch_row(static_cast<const uint8_t*>(p.r) + o, p.c, lane);
          else prefetch_row(static_cast<const TS*>(p.r) + o, p.c, lane);
        }
        if (p.dgate != nullptr && p.u_e == nullptr) prefetch_row(static_cast<const TC*>(p.u) + o, p.c, lane);
        if (OWN && gated) prefetch_row(gate - ch + ahead.row * p.gate_ld, p.c, lane);
        if (OWN && adaptive) prefetch_row(gs - ch + ahead.row * p.gate_shift_ld, p.c, lane);
      }
    }
    const uint4* s = ring + stage * p.slots * kRowThreads;
    const long long o = static_cast<long long>(here.row) * p.c + ch, e = static_cast<long long>(here.row) * groups;
    int k[P];                                // channels that are there
#pragma unroll
    for (int q = 0; q < P; ++q) k[q] = row_there ? inside[q] : 0;
    // All pieces of a tensor, or of its rows in 8 bits.  is_r: it is r, whose exponents are in r_ex; others read theirs.  (Slots do not tell r from others: what is not there
    // takes none.)  (A question that is the same for all pieces is asked once: the pieces' instructions then lie side by side.)
    auto take = [&](auto tag, auto is_r, int slot, const void* t, const uint8_t* exponents, Pairs (&v)[P]) {
      using E = decltype(tag);
      constexpr bool kIsR = decltype(is_r)::value;
      if (exponents == nullptr) {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          if constexpr (VEC) v[q] = ring_take<E>(s + (slot + q * (static_cast<int>(sizeof(E)) / 2)) * kRowThreads);
          else v[q] = load_piece<E, VEC>(static_cast<const E*>(t) + o + q * kStep, k[q]);
        }
      } else if (VEC && (kIsR || p.words)) {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const uint4 w = s[(slot + q) * kRowThreads];
          uint32_t ex = w.z >> (ch + q * kStep) / kGroup8 % 4 * 8 & 255u;
          if constexpr (kIsR) ex = p.words ? ex : r_ex[q];
          v[q] = values8(make_uint2(w.x, w.y), ex);
        }
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) v[q] = load_piece8<VEC>(static_cast<const uint8_t*>(t) + o + q * kStep, exponents + e + (ch + q * kStep) / kGroup8, k[q]);
      }
    };
    // gates (gate_at) of this row's output, or of its norm
    auto own_gates = [&](const TC* row, int slot, int q) {
      Pairs t;
      if constexpr (VEC) t = ring_take<TC>(s + (slot + q * kC) * kRowThreads);
      else t = load_piece<TC, VEC>(row + q * kStep, k[q]);
      return each(t, [](float a) { return gate_at<TC>(a); });
    };
    if (!OWN && here.at == 0) {
      const unsigned gate_row = here.gate_row(p.plan);
      auto opened = [](float a) { return open_of(gate_at<TC>(a)); };
      if (gated) {
#pragma unroll
        for (int q = 0; q < P; ++q) open[OWN ? 0 : q] = each(load_piece<TC, VEC>(gate + gate_row * p.gate_ld + q * kStep, k[q]), opened);
      }
      if (adaptive) {
#pragma unroll
        for (int q = 0; q < P; ++q) m[q] = each(load_piece<TC, VEC>(gs + gate_row * p.gate_shift_ld + q * kStep, k[q]), opened);
      }
    }
    Pairs t[P];
    if (p.norm != kNoNorm) {
      Pairs z[P], g[P], d[P];
      take(TS{}, std::true_type{}, p.s_r, p.r, p.r_e, z);
      take(TC{}, std::false_type{}, p.s_dy, p.dy, nullptr, d);
      if (OWN && adaptive) {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          m[q] = own_gates(gs + here.row * p.gate_shift_ld, p.s_g, q);
          g[q] = mul(d[q], each(m[q], [](float a) { return open_of(a); }));
        }
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) g[q] = mul(d[q], m[q]);
      }
      Pairs sz = z[0], sg = g[0];
#pragma unroll
      for (int q = 1; q < P; ++q) {
        sz = add(sz, z[q]);
        sg = add(sg, g[q]);
      }
      float sums[2] = {total(sz), total(sg)};
      team_sum<LANES>(sums);
      const float mean = sums[0] * inv_c;
      const Pairs minus_mean_g = both(-sums[1] * inv_c);
      sz = sg = both(0.f);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        z[q] = add(z[q], both(inside[q] > 0 ? -mean : 0.f));      // (nothing stays nothing)
        if constexpr (!VEC) {
#pragma unroll
          for (int i = 0; i < kPiece; ++i)
            if (i >= inside[q]) z[q].v[i / 2] = i & 1 ? ptx::pack2(z[q].get(i - 1), 0.f) : ptx::pack2(0.f, 0.f);
        }
        sz = fma(z[q], z[q], sz);
        sg = fma(g[q], z[q], sg);
      }
      sums[0] = total(sz);
      sums[1] = total(sg);
      team_sum<LANES>(sums);
      const float rstd = row_there ? rsqrtf(fmaf(sums[0], inv_c, p.eps)) : 0.f;      // (no row: no number where eps is zero)
      const Pairs rstd2 = both(rstd), minus_mean_gz = both(-sums[1] * inv_c * rstd);
#pragma unroll
      for (int q = 0; q < P; ++q) {
        z[q] = mul(z[q], rstd2);
        t[q] = mul(rstd2, fma(z[q], minus_mean_gz, add(g[q], minus_mean_g)));
      }
      if constexpr (VEC && P > 1) take(TC{}, std::false_type{}, p.s_dy, p.dy, nullptr, d);               // (read again: it frees the registers meanwhile)
      if (OWN && adaptive) {
        if (p.dgate_shift != nullptr) {
          TC* to = static_cast<TC*>(p.dgate_shift) + 2 * (o - ch) + ch;
#pragma unroll
          for (int q = 0; q < P; ++q) {
            store_piece<VEC>(to + q * kStep, mul(mul(d[q], z[q]), each(m[q], [](float a) { return slope_of(a); })), k[q]);
            store_piece<VEC>(to + p.c + q * kStep, d[q], k[q]);
          }
        }
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          a0[kSums ? q : 0] = fma(d[q], z[q], a0[kSums ? q : 0]);
          a1[kSums ? q : 0] = add(a1[kSums ? q : 0], d[q]);
        }
      }
      if (p.dr != nullptr) {
        take(TS{}, std::false_type{}, 0, p.dr, nullptr, z);
#pragma unroll
        for (int q = 0; q < P; ++q) t[q] = add(t[q], z[q]);
      }
    } else {
      take(TS{}, std::false_type{}, 0, p.dr, nullptr, t);
    }
    if (p.dgate != nullptr) {
      Pairs u[P];
      take(TC{}, std::false_type{}, p.s_u, p.u, p.u_e, u);
      if constexpr (OWN) {
        TC* to = static_cast<TC*>(p.dgate) + o;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const Pairs own = own_gates(gate + here.row * p.gate_ld, p.s_gate, q);
          store_piece<VEC>(to + q * kStep, mul(mul(t[q], u[q]), each(own, [](float a) { return slope_of(a); })), k[q]);
          if (p.du != nullptr) store_piece<VEC>(static_cast<TC*>(p.du) + o + q * kStep, mul(t[q], each(own, [](float a) { return open_of(a); })), k[q]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) a2[OWN ? 0 : q] = fma(t[q], u[q], a2[OWN ? 0 : q]);
      }
    }
    if (p.du != nullptr && !(OWN && p.dgate != nullptr)) {
      TC* to = static_cast<TC*>(p.du) + o;
      if (OWN && gated) {
#pragma unroll
        for (int q = 0; q < P; ++q)
          store_piece<VEC>(to + q * kStep, mul(t[q], each(own_gates(gate + here.row * p.gate_ld, p.s_gate, q), [](float a) { return open_of(a); })), k[q]);
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) store_piece<VEC>(to + q * kStep, OWN ? t[q] : mul(t[q], open[OWN ? 0 : q]), k[q]);
      }
    }
    if (p.x != nullptr) {
      Pairs x[P];
      if (VEC && GATES == kOwnAdaptive && P == 4 && sizeof(TC) == 4 && p.s_x < 0) {
#pragma unroll
        for (int q = 0; q < P; ++q)
          x[q] = p.x_e != nullptr ? load_piece8<VEC>(static_cast<const uint8_t*>(p.x) + o + q * kStep, p.x_e + e + (ch + q * kStep) / kGroup8, k[q])
                                  : load_piece<TS, VEC>(static_cast<const TS*>(p.x) + o + q * kStep, k[q]);
      } else {
        take(TS{}, std::false_type{}, p.s_x, p.x, p.x_e, x);
      }
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const Pairs v = mul(t[q], x[q]);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) scale_sums[(q * kPiece + i) * kRowThreads] += v.get(i);
      }
    }
    if (p.dx != nullptr) {
      if (p.scale != nullptr) {
#pragma unroll
        for (int q = 0; q < P; ++q) t[q] = mul(t[q], vector(p.scale, q, 0.f));
      }
      TS* to = static_cast<TS*>(p.dx) + o;
#pragma unroll
      for (int q = 0; q < P; ++q) store_piece<VEC>(to + q * kStep, t[q], k[q]);
    }
    if constexpr (!OWN) {
      if (here.at + 1 == p.plan.chunk) {
        // the end of a piece: the gates' gradients from the sums over their samples, the logits once more for their slopes; or the sums for the second kernel
        const bool there = here.unit < p.plan.units;
        const unsigned gate_row = here.gate_row(p.plan);
        auto slope = [](float a) { return slope_of(gate_at<TC>(a)); };
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          // the norm's gates and shifts, the output gate
          if (which == 0 ? !adaptive : p.dgate == nullptr) continue;
#pragma unroll
          for (int q = 0; q < P; ++q) {
            const int n = there ? inside[q] : 0;
            if (p.pieces != nullptr) {
              float* d = p.pieces + static_cast<long long>(there ? here.unit : 0) * 3 * p.c + ch + q * kStep;
              if (which == 0) {
                store_piece<VEC>(d, a0[q], n);
                store_piece<VEC>(d + p.c, a1[q], n);
              } else {
                store_piece<VEC>(d + 2 * p.c, a2[OWN ? 0 : q], n);
              }
            } else if (which == 1) {
              store_piece<VEC>(static_cast<TC*>(p.dgate) + static_cast<long long>(gate_row) * p.c + ch + q * kStep,
                               mul(a2[OWN ? 0 : q], each(load_piece<TC, VEC>(gate + gate_row * p.gate_ld + q * kStep, n), slope)), n);
            } else if (p.dgate_shift != nullptr) {
              TC* d = static_cast<TC*>(p.dgate_shift) + static_cast<long long>(gate_row) * 2 * p.c + ch + q * kStep;
              store_piece<VEC>(d, mul(a0[q], each(load_piece<TC, VEC>(gs + gate_row * p.gate_shift_ld + q * kStep, n), slope)), n);
              store_piece<VEC>(d + p.c, a1[q], n);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < P; ++q) {
          a2[OWN ? 0 : q] = both(0.f);
          if (adaptive) a0[q] = a1[q] = both(0.f);
        }
      }
    }
    here.next(p.plan, team, step);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
  }

  if (p.partial != nullptr) {
    // the block's teams in their order; the ring's memory, in which nothing is on its way any more
    copy_async_wait<0>();
    constexpr int kAll = kRowThreads / LANES, kWidth = LANES * P * kPiece;
    float* flat = reinterpret_cast<float*>(ring_memory);      // [team][kWidth]
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      if (j == 2 && p.x == nullptr) break;
      __syncthreads();
#pragma unroll
      for (int q = 0; q < P; ++q)
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
          flat[static_cast<int>(threadIdx.x) / LANES * kWidth + ch + q * kStep + i * channel_step<VEC>()] =
              j == 2 ? scale_sums[(q * kPiece + i) * kRowThreads] : !kSums ? 0.f : (j == 0 ? a0 : a1)[kSums ? q : 0].get(i);
      __syncthreads();
      for (int i = threadIdx.x; i < p.c; i += kRowThreads) {
        float t = 0.f;
#pragma unroll 4
        for (int q = 0; q < kAll; ++q) t += flat[q * kWidth + i];
        p.partial[(static_cast<long long>(blockIdx.x) * 3 + j) * p.c + i] = t;
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
      v = s[0] * slope_of(gate_at<TC>(static_cast<float>(gs[row * gs_ld + ch])));
      store_vec<1>(d, &v);
      store_vec<1>(d + c, &s[1]);
    }
    if (dgate != nullptr) {
      v = s[2] * slope_of(gate_at<TC>(static_cast<float>(gate[row * gate_ld + ch])));
      store_vec<1>(dgate + static_cast<long long>(row) * c + ch, &v);
    }
  }
}

// Blocks of an SM, at most, and SMs: the workspace is sized by them.
constexpr int most_blocks(int c) { return c <= 256 ? 6 : 3; }
constexpr int kMostSms = 160;
// Pieces of gate rows' samples, at most: two for each team that is at work (row_plan).
constexpr long long most_units(int c) { return 2ll * kMostSms * most_blocks(c) * (c <= 128 ? 16 : c <= 384 ? 8 : 4); }

struct Sums {
  float *dweight, *dbias, *dscale;
};

template <typename TS, typename TC, int LANES, int P, bool VEC, int GATES>
int launch(cudaStream_t stream, GradParams p, const Sums& sums, long long rows, int samples, int l) {
  constexpr bool OWN = GATES != kSharedGates;
  constexpr auto kernel = residual_norm_grad_kernel<TS, TC, LANES, P, VEC, GATES>;
  constexpr int kS = P * sizeof(TS) / 2, kC = P * sizeof(TC) / 2, kWarps = kRowThreads / 32, kTeams = 32 / LANES, kFlat = kRowThreads * P * kPiece * 4;
  static std::once_flag once;
  static int held = 1;
  std::call_once(once, [&] {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, kRowThreads, 0) != cudaSuccess) cudaGetLastError();
    held = held < 1 ? 1 : held;
  });
  // (a row in 8 bits takes one slot a piece)
  int slots = p.dr != nullptr ? kS : 0;
  auto place = [&](bool there, bool small, int size) {
    const int at = slots;
    slots += !there ? 0 : small ? P : size;
    return at;
  };
  p.s_dy = place(p.norm != kNoNorm, false, kC);
  p.s_r = place(p.norm != kNoNorm, p.r_e != nullptr, kS);
  p.s_u = place(p.dgate != nullptr, p.u_e != nullptr, kC);
  p.s_gate = place(OWN && p.gate != nullptr, false, kC);
  p.s_g = place(OWN && p.gate_shift != nullptr, false, kC);
  // (seven float32 tensors of more than 768 channels, or six and x in 8 bits, are more than the ring holds)
  constexpr int kStage = VEC ? depth<TS, TC, P, OWN>() * kRowThreads * 16 : 0;
  p.s_x = p.x != nullptr && (slots + (p.x_e != nullptr ? P : kS)) * kStage + kFlat > kMostRing ? -1 : place(p.x != nullptr, p.x_e != nullptr, kS);
  p.slots = slots;
  int smem = slots * kStage;
  if (p.partial != nullptr && smem < kFlat) smem = kFlat;
  p.s_scale = smem / 16 / kRowThreads;
  if (p.x != nullptr) smem += kFlat;
  KFB_TRY(allow_smem<kernel>(kMostRing));
  KFB_CHECK_ARG(smem <= kMostRing, "residual_norm_bwd: %d bytes of shared memory", smem);
  const int fit = smem > 0 ? kMostRing / smem : held, limit = held < most_blocks(p.c) ? held : most_blocks(p.c), blocks_per_sm = limit < fit ? limit : fit;
  const long long most = static_cast<long long>(sm_count() < kMostSms ? sm_count() : kMostSms) * blocks_per_sm;
  const bool gates = p.dgate != nullptr || p.dgate_shift != nullptr;
  p.plan = row_plan(rows, samples, l, most * kWarps * kTeams, kTeams, gates ? 2 * 3 * 4 * p.c : 0);
  if (p.plan.chunks == 1 || !gates) p.pieces = nullptr;
  else KFB_CHECK_ARG(p.plan.units <= most_units(p.c), "residual_norm_bwd: %u pieces", p.plan.units);
  const long long want = (p.plan.sets + kWarps - 1) / kWarps;
  const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
  {
    LaunchScope scope(stream, "residual_norm_grad");
    KFB_TRY(launch_kernel(stream, kernel, blocks, kRowThreads, smem, p));
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
    KFB_TRY(launch_kernel(stream, residual_norm_sum_kernel, cdiv((p.x != nullptr ? 3 : 2) * p.c, 32), 1024, 0, const_cast<const float*>(p.partial), sums.dweight,
                          sums.dbias, sums.dscale, static_cast<int>(blocks), p.c));
  }
  return KFB_OK;
}

template <typename TS, typename TC, int LANES, int P, bool VEC>
int launch_own(cudaStream_t stream, const GradParams& p, const Sums& sums, long long rows, int samples, int l) {
  if (samples > 1) return launch<TS, TC, LANES, P, VEC, kSharedGates>(stream, p, sums, rows, samples, l);
  return p.norm == kAdaptiveNorm ? launch<TS, TC, LANES, P, VEC, kOwnAdaptive>(stream, p, sums, rows, samples, l)
                                 : launch<TS, TC, LANES, P, VEC, kOwnGates>(stream, p, sums, rows, samples, l);
}

template <typename TS, typename TC>
int dispatch(cudaStream_t stream, GradParams p, const Sums& sums, long long rows, int samples, int l) {
  auto of = [](const void* q, const uint8_t* e) { return reinterpret_cast<uintptr_t>(q) << (e != nullptr ? 1 : 0); };   // bytes: 8-byte boundaries do
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.dr) | reinterpret_cast<uintptr_t>(p.dy) | of(p.r, p.r_e) | of(p.u, p.u_e) | of(p.x, p.x_e) |
                       reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.gate_shift) | reinterpret_cast<uintptr_t>(p.dx) |
                       reinterpret_cast<uintptr_t>(p.du) | reinterpret_cast<uintptr_t>(p.dgate) | reinterpret_cast<uintptr_t>(p.dgate_shift) |
                       static_cast<uintptr_t>((p.gate_ld | p.gate_shift_ld) * sizeof(TC));
  p.words = groups8(p.c) % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.r_e) | reinterpret_cast<uintptr_t>(p.u_e) | reinterpret_cast<uintptr_t>(p.x_e)) & 3) == 0;
#define KFB_CALL(LANES, P, VEC) launch_own<TS, TC, LANES, P, VEC>(stream, p, sums, rows, samples, l)
  KFB_ROW_SHAPES(p.c, p.c % 8 == 0 && (at & 15) == 0, KFB_CALL);
#undef KFB_CALL
}

size_t partial_bytes(int c) { return align_up(static_cast<size_t>(kMostSms) * most_blocks(c) * 3 * c * sizeof(float), 256); }

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
