// A linear layer's products with what follows them, many rows, bf16:
//   forward   out = f(a b^T + bias) + aux        backward   out = aux f'(a b^T + bias), and sums of it over rows        plain   out = a b^T
//
// What bounds it: a in and out out, HBM, and the element-wise tail: an output's f' takes 20 to 30 instructions, as long as the products of 512 channels with it.
// Split: a CTA pair (cta_group::2) takes tiles of 256 rows by BN columns, one column tile throughout, so that the sums over rows stay in registers from tile to
// tile.  A thread fetches operands into a ring, a thread of the even CTA issues the products into one of two accumulators; two groups of eight warps take the
// tiles in turn.  A group has a buffer for its tile: aux comes into it through TMA while the other group works, is worked on in place, and the buffer
// leaves through TMA; a thread of its own sees to both.
// 147 456 rows, 512 -> 256 with gelu: forward 50 us (0.77 PFLOP/s, 4.5 TB/s; 55 % of the issue slots are the tail's), gradient of z 62 us, dx 43 us (writes alone
// reach 4 TB/s); 18 432 rows, 384 -> 1 536: forward 22 us (1.0 PFLOP/s), what the library's product without bias takes.
// The operand b is read as it lies, along k (the forward pass) or across it (dx = dz W).
#include <mutex>

#include "gemm.cuh"   // pack_bf16x2
#include "linear_tail.cuh"
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int kRows = 128;                           // of a CTA
constexpr int kBox = kRows * 128;                    // [128 rows][64 columns], 128-byte swizzle
constexpr int kRowsBox = 64 * 128;                   // [64 k][64 columns] of b across k
constexpr int kTailWarp = 4, kGroupWarps = 8;
constexpr int kThreads = 32 * (kTailWarp + 2 * kGroupWarps);

template <int BN>
struct Cfg {
  static constexpr int kBBoxes = (BN / 2 + 63) / 64;                  // of 64 columns, across k
  static constexpr int kBStage = kBBoxes * kRowsBox, kStage = kBox + kBStage;
  static constexpr int kBBytes = BN / 2 * 128;       // along k: what comes
  static constexpr int kPasses = BN / 64;            // a group has 64 columns in a buffer at a time, of which a warp has 32
  static constexpr int kFit = (232448 - 1536 - BN * 4 - 4 * kBox) / kStage, kStages = kFit < 6 ? kFit : 6;
  static constexpr int kTmem = BN == 128 ? 256 : 512;
  static constexpr int kSmem = kStages * kStage + 4 * kBox + BN * 4 + 512 + 1024;
  static_assert(BN % 64 == 0 && kStages >= 3, "tiles of 128, 192 or 256 columns");
  static_assert(kSmem <= 232448, "shared memory");
};

struct PairParams {
  int rows, n, blocks, row_blocks, n_tiles, groups;  // blocks of 64 along k; pairs that share a column tile
  const float* bias;
  int act, has_aux;
  float* partial;
};

// The warps of both groups.
__device__ __forceinline__ void tail_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(64 * kGroupWarps) : "memory"); }

template <int BN, int TAIL, bool BY_K>
__global__ void __launch_bounds__(kThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_aux,
                   const __grid_constant__ CUtensorMap tm_out, const PairParams p) {
  using K = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tiles = ring + K::kStages * K::kStage;
  float* s_bias = reinterpret_cast<float*>(tiles + 4 * kBox);              // of the tile's columns
  uint64_t* full = reinterpret_cast<uint64_t*>(s_bias + BN);               // in the leader: both CTAs' copies
  uint64_t* empty = full + K::kStages;
  uint64_t* acc_full = empty + K::kStages;           // [2]
  uint64_t* acc_empty = acc_full + 2;                // [2], in the leader: the group's warps in both CTAs
  uint64_t* ready = acc_empty + 2;                   // [group][buffer] aux has come, or the buffer is free
  uint64_t* done = ready + 4;                        // [group][buffer] the group's warps have written it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int pair = blockIdx.x >> 1, first = pair / p.n_tiles, n0 = pair % p.n_tiles * BN;
  const int my_tiles = first < p.row_blocks ? (p.row_blocks - first + p.groups - 1) / p.groups : 0;
  auto row0_of = [&](int i) { return (2 * (first + i * p.groups) + rank) * kRows; };

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tm_a);
    ptx::prefetch_tmap(&tm_b);
    ptx::prefetch_tmap(&tm_out);
    for (int i = 0; i < K::kStages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&acc_full[i], 1);
      ptx::mbar_init(&acc_empty[i], 2 * kGroupWarps);
    }
    for (int i = 0; i < 4; ++i) {
      ptx::mbar_init(&ready[i], 1);
      ptx::mbar_init(&done[i], kGroupWarps);
    }
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, K::kTmem);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before_sync();
  __syncwarp();
  ptx::cluster_sync();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_enter();

  if (warp == 0) {
    if (ptx::elect_one()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i)
        for (int kb = 0; kb < p.blocks; ++kb) {
          ok = ptx::mbar_wait(&empty[st], ph ^ 1, 701);
          if (!ok) break;
          if (rank == 0) ptx::mbar_expect_tx(&full[st], 2 * (kBox + (BY_K ? K::kBStage : K::kBBytes)));
          const uint32_t bar = ptx::leader_addr(&full[st]);
          uint8_t *a = ring + st * K::kStage, *b = a + kBox;
          ptx::tma_load_4d_pair(a, &tm_a, bar, kb * 64, row0_of(i), 0, 0);
          if constexpr (BY_K) {
#pragma unroll
            for (int q = 0; q < K::kBBoxes; ++q) ptx::tma_load_4d_pair(b + q * kRowsBox, &tm_b, bar, n0 + rank * (BN / 2) + q * 64, kb * 64, 0, 0);
          } else {
            ptx::tma_load_4d_pair(b, &tm_b, bar, kb * 64, n0 + rank * (BN / 2), 0, 0);
          }
          if (++st == K::kStages) { st = 0; ph ^= 1u; }
        }
      for (int i = 0; ok && i < K::kStages; ++i) {     // the last products' arrivals at this CTA's barriers, before it may exit
        ok = ptx::mbar_wait(&empty[st], ph ^ 1, 702);
        if (++st == K::kStages) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && ptx::elect_one()) {
      constexpr uint32_t idesc = ptx::make_idesc(2 * kRows, BN, 1) | (BY_K ? 1u << 16 : 0u);
      constexpr uint32_t b_step = BY_K ? 2048 >> 4 : 2;      // of 16 k
      const uint64_t a0 = ptx::make_kmajor_desc<128>(ptx::smem_u32(ring));
      // across k: rows of 128 bytes, one per k; eight of them 1024 bytes apart, the next 64 columns a box further
      const uint64_t b0 = BY_K ? static_cast<uint64_t>((ptx::smem_u32(ring + kBox) & 0x3ffff) >> 4) | (static_cast<uint64_t>(kRowsBox >> 4) << 16) |
                                     (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61)
                               : ptx::make_kmajor_desc<128>(ptx::smem_u32(ring + kBox));
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int i = 0; ok && i < my_tiles; ++i) {
        const int g = i & 1;
        ok = ptx::mbar_wait(&acc_empty[g], (i >> 1 & 1) ^ 1, 703, ptx::kPolls);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        for (int kb = 0; kb < p.blocks; ++kb) {
          ok = ptx::mbar_wait(&full[st], ph, 704, ptx::kPolls);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const uint64_t a = a0 + st * (K::kStage >> 4), b = b0 + st * (K::kStage >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) ptx::mma_f16_ss_pair(tmem + g * BN, a + k * 2, b + k * b_step, idesc, kb > 0 || k > 0 ? 1u : 0u);
          ptx::tc_commit_pair(&empty[st]);
          if (++st == K::kStages) { st = 0; ph ^= 1u; }
        }
        if (ok) ptx::tc_commit_pair(&acc_full[g]);
      }
    }
  } else if (warp < kTailWarp) {
    // ---------------------------------------------------------------- a group's buffer: aux in, the tile out
    if (ptx::elect_one()) {
      const int g = warp - 2;
      const int count = (my_tiles - g + 1) / 2 * K::kPasses;      // passes of the group's tiles
      auto row0_at = [&](int q) { return row0_of(g + q / K::kPasses * 2); };
      auto arm = [&](int q) {
        uint64_t* bar = &ready[2 * g + (q & 1)];
        if (TAIL != kPlainTail && p.has_aux) {
          ptx::mbar_expect_tx(bar, kBox);
          ptx::tma_load_4d(tiles + (2 * g + (q & 1)) * kBox, &tm_aux, bar, n0 + q % K::kPasses * 64, row0_at(q), 0, 0);
        } else {
          ptx::mbar_arrive(bar);
        }
      };
      for (int q = 0; q < 2 && q < count; ++q) arm(q);
      for (int q = 0; q < count; ++q) {
        if (!ptx::mbar_wait(&done[2 * g + (q & 1)], q >> 1 & 1, 705)) break;
        const int col = n0 + q % K::kPasses * 64;
        if (row0_at(q) < p.rows && col < p.n) {
          ptx::tma_store_4d(&tm_out, tiles + (2 * g + (q & 1)) * kBox, col, row0_at(q), 0, 0);
          ptx::tma_store_commit();
        }
        if (q + 2 < count) {
          ptx::tma_store_wait_read();                // (the group has the other buffer meanwhile)
          arm(q + 2);
        }
      }
      ptx::tma_store_wait_all();
    }
  } else {
    // ---------------------------------------------------------------- the tail: a warp has 32 rows (tensor-memory lanes) of half of the columns
    const int g = (warp - kTailWarp) / kGroupWarps, quad = warp & 3, half = (warp - kTailWarp) / 4 % 2, r = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + g * BN + half * 32;
    uint8_t* row = tiles + 2 * g * kBox + r * 128;
    float sums[K::kPasses];                          // of column 8 (lane & 3) + what sum_rows8 gives, of each pass
#pragma unroll
    for (int j = 0; j < K::kPasses; ++j) sums[j] = 0.f;
    if constexpr (TAIL != kPlainTail) {
      for (int c = threadIdx.x - 32 * kTailWarp; c < BN; c += 64 * kGroupWarps) s_bias[c] = p.bias != nullptr && n0 + c < p.n ? p.bias[n0 + c] : 0.f;
      tail_barrier();
    }
    bool ok = true;
    int at_pass = 0;
    for (int i = g; ok && i < my_tiles; i += 2) {
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&acc_full[g], i >> 1 & 1, 707)) != 0;
      if (!ok) break;
      ptx::tc_fence_after_sync();
#pragma unroll 1                                      // (unrolled, the code of four passes does not stay in the instruction caches)
      for (int pass = 0; pass < K::kPasses; ++pass, ++at_pass) {
        const int buffer = at_pass & 1, col = pass * 64 + half * 32;
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&ready[2 * g + buffer], at_pass >> 1 & 1, 706)) != 0;
        if (!ok) break;
        uint32_t raw[32];
        ptx::tmem_ld_32x32b_x32(t_row + pass * 64, raw);
        ptx::tmem_ld_wait();
        if (pass + 1 == K::kPasses) {
          ptx::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(ptx::leader_addr(&acc_empty[g]));
        }
        auto cell_at = [&](int c) { return reinterpret_cast<uint4*>(row + buffer * kBox + ((half * 4 + c) ^ (r & 7)) * 16); };
        if constexpr (TAIL == kPlainTail) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = pack_bf16x2(__uint_as_float(raw[8 * c + 2 * q]), __uint_as_float(raw[8 * c + 2 * q + 1]));
            *cell_at(c) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          float mine = 0.f;
          with_activation(p.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint64_t v[4], x[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) v[q] = ptx::pack2(raw[8 * c + 2 * q], raw[8 * c + 2 * q + 1]);
              const ulonglong2* b = reinterpret_cast<const ulonglong2*>(s_bias + col + 8 * c);
              const ulonglong2 lo = b[0], hi = b[1];
              v[0] = ptx::add2(v[0], lo.x), v[1] = ptx::add2(v[1], lo.y), v[2] = ptx::add2(v[2], hi.x), v[3] = ptx::add2(v[3], hi.y);
              uint4* cell = cell_at(c);
              if (TAIL == kBackwardTail || p.has_aux) {
                const uint4 a = *cell;
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q] = ptx::pack2(aw[q] << 16, aw[q] & 0xffff0000u);
              }
              if constexpr (TAIL == kForwardTail) {
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = activation<ACT>(v[q]);
                if (p.has_aux) {
#pragma unroll
                  for (int q = 0; q < 4; ++q) v[q] = ptx::add2(v[q], x[q]);
                }
              } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = ptx::mul2(x[q], slope<ACT>(v[q]));
                if (p.partial != nullptr) {
                  const float s = sum_rows8(v, lane);
                  if ((lane & 3) == c) mine = s;
                }
              }
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) w[q] = pack_bf16x2(v[q]);
              *cell = make_uint4(w[0], w[1], w[2], w[3]);
            }
          });
#pragma unroll
          for (int j = 0; j < K::kPasses; ++j) sums[j] += j == pass ? mine : 0.f;
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&done[2 * g + buffer]);
      }
    }
    if (TAIL == kBackwardTail && p.partial != nullptr) {
      // a row of partial sums for each CTA of a column tile: its warps' through the ring, whose operands the last product has read
      float* warps = reinterpret_cast<float*>(ring);      // [group, quadrant][BN]
      tail_barrier();
#pragma unroll
      for (int j = 0; j < K::kPasses; ++j)
        warps[(g * 4 + quad) * BN + j * 64 + half * 32 + 8 * (lane & 3) + 4 * (lane >> 4 & 1) + 2 * (lane >> 3 & 1) + (lane >> 2 & 1)] = sums[j];
      tail_barrier();
      const int c = threadIdx.x - 32 * kTailWarp;
      if (c < BN && n0 + c < p.n) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += warps[w * BN + c];
        p.partial[static_cast<long long>(first * 2 + rank) * p.n + n0 + c] = s;
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncwarp();
  ptx::cluster_sync();      // neither CTA leaves while the other may still read its operands or reach its barriers
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem, K::kTmem);
  }
}

template <int BN, int TAIL, bool BY_K>
int pairs_held() {
  static std::once_flag once[64];
  static int held[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::call_once(once[dev & 63], [&] { held[dev & 63] = clusters_held(linear_pair_kernel<BN, TAIL, BY_K>, 2, kThreads, Cfg<BN>::kSmem); });
  return held[dev & 63];
}

// A tile's columns: 256, or 192 or 128 where these leave fewer of them unused (63 001 rows, 1 536 -> 384: by 192 66 us, by 256 74; 128 -> 128: by 128 11, by 256 17).
int tile_width(int n) {
  int best = 256;
  for (int w : {192, 128})
    if (cdiv(n, w) * w < cdiv(n, best) * best) best = w;
  return best;
}

struct Grid {
  int bn, n_tiles, row_blocks, groups;
};
Grid grid_of(long long rows, int n, int held) {
  Grid g;
  g.bn = tile_width(n);
  g.n_tiles = cdiv(n, g.bn);
  g.row_blocks = static_cast<int>((rows + 2 * kRows - 1) / (2 * kRows));
  g.groups = held / g.n_tiles;
  if (g.groups > g.row_blocks) g.groups = g.row_blocks;
  return g;
}

int matrix_map(CUtensorMap* m, const void* ptr, long long rows, long long cols, int box_rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1, 1};
  const uint64_t str[3] = {static_cast<uint64_t>(cols) * 2, static_cast<uint64_t>(cols) * 2 * rows, static_cast<uint64_t>(cols) * 2 * rows};
  const uint32_t box[4] = {64, static_cast<uint32_t>(box_rows), 1, 1};
  return make_tmap(m, ptr, 2, 4, dims, str, box, 128);
}

template <int BN, int TAIL, bool BY_K>
int launch_as(cudaStream_t stream, const LinearPair& q, const char* tag) {
  const int held = pairs_held<BN, TAIL, BY_K>();
  const Grid g = grid_of(q.rows, q.n, held);
  KFB_CHECK_ARG(held > 0 && g.groups > 0, "linear: the device holds no pair of this kernel");
  CUtensorMap ta, tb, tx, to;
  KFB_TRY(matrix_map(&ta, q.a, q.rows, q.k, kRows));
  if (BY_K) KFB_TRY(matrix_map(&tb, q.b, q.k, q.n, 64));
  else KFB_TRY(matrix_map(&tb, q.b, q.n, q.k, BN / 2));
  KFB_TRY(matrix_map(&to, q.out, q.rows, q.n, kRows));
  tx = to;
  if (q.aux != nullptr) KFB_TRY(matrix_map(&tx, q.aux, q.rows, q.n, kRows));
  PairParams p = {};
  p.rows = static_cast<int>(q.rows);
  p.n = q.n;
  p.blocks = cdiv(q.k, 64);
  p.row_blocks = g.row_blocks;
  p.n_tiles = g.n_tiles;
  p.groups = g.groups;
  p.bias = q.bias;
  p.act = q.act;
  p.has_aux = q.aux != nullptr;
  p.partial = q.partial;
  LaunchScope scope(stream, tag);
  return launch_kernel_clustered(stream, linear_pair_kernel<BN, TAIL, BY_K>, 2, 2 * g.n_tiles * g.groups, kThreads, Cfg<BN>::kSmem, ta, tb, tx, to, p);
}

template <int BN>
int launch_width(cudaStream_t stream, const LinearPair& q, const char* tag) {
  if (q.tail == kForwardTail) return launch_as<BN, kForwardTail, false>(stream, q, tag);
  if (q.tail == kBackwardTail) return launch_as<BN, kBackwardTail, false>(stream, q, tag);
  return launch_as<BN, kPlainTail, true>(stream, q, tag);
}

int backward_pairs(int n) {
  const int w = tile_width(n);
  return w == 256 ? pairs_held<256, kBackwardTail, false>() : w == 192 ? pairs_held<192, kBackwardTail, false>() : pairs_held<128, kBackwardTail, false>();
}

}  // namespace

// Half of the pairs at least have a tile.  By pairs and by tiles of 128 x 64 (matmul.cu), silu: 4 096 rows, 768 -> 768 (48 pairs of 74) 12 and 17 us; 2 048 rows, 384 -> 1 536
// (48) 10 and 14; 8 192 rows, 512 -> 256 (32) 10 and 9; 4 096 rows (16) 10 and 6.6.
bool linear_pair_ok(long long rows, int n, int k) {
  const int held = backward_pairs(n);
  if (held <= 0 || n < 64 || k < 64) return false;
  const Grid g = grid_of(rows, n, held);
  return g.groups > 0 && 2 * g.groups * g.n_tiles >= held;
}

int linear_pair_partials(long long rows, int n) { return grid_of(rows, n, backward_pairs(n)).groups * 2; }

int launch_linear_pair(cudaStream_t stream, const LinearPair& p, const char* tag) {
  KFB_CHECK_ARG((p.tail == kPlainTail) == (p.by_k != 0), "linear: tail %d with an operand %s k", p.tail, p.by_k ? "across" : "along");
  const int w = tile_width(p.n);
  return w == 256 ? launch_width<256>(stream, p, tag) : w == 192 ? launch_width<192>(stream, p, tag) : launch_width<128>(stream, p, tag);
}

}  // namespace kfb
