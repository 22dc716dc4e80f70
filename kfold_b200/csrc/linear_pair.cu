// A linear layer's products with what follows them, many rows, bf16:
//   forward   out = f(a b^T + bias) + aux        backward   out = aux f'(a b^T + bias), and sums of it over rows        plain   out = a b^T
//
// What bounds it: a in and out out, HBM, and the element-wise tail: an output's f' takes 20 to 30 instructions, as long as the products of 512 channels with it.
// Split: a CTA pair (cta_group::2) takes tiles of 256 rows by BN columns, one column tile throughout, so that the sums over rows stay in registers from tile to
// tile.  A thread fetches operands into a ring, a thread of the even CTA issues the products into one of two accumulators; two groups of eight warps take the
// tiles in turn.  A group has a buffer for its tile: aux comes into it through TMA while the other group works, is worked on in place, and the buffer
// leaves through TMA; a thread of its own sees to both.
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
  static constexpr int kBStage = BN / 2 * 128, kStage = kBox + kBStage;
  static constexpr int kTile = BN / 64 * kBox;       // a group's buffer
  static constexpr int kStages = BN == 256 ? 3 : 6;
  static constexpr int kSmem = kStages * kStage + 2 * kTile + 512 + 1024;
  static constexpr int kChunks = BN / 64;            // 32-column chunks of a warp: half of the tile's columns
  static_assert(kSmem <= 232448, "shared memory");
};

struct PairParams {
  int rows, n, blocks, row_blocks, n_tiles, groups;  // blocks of 64 along k; pairs that share a column tile
  const float* bias;
  int act, has_aux;
  float* partial;
};

// Sums over a warp's rows (lanes) of eight columns: lane l has column 4 (l >> 4 & 1) + 2 (l >> 3 & 1) + (l >> 2 & 1) at the end.  (Half of the columns change hands
// at each of the first three steps.)
__device__ __forceinline__ float sum_rows(const float (&v)[8], int lane) {
  float a[4], b[2];
  const bool h4 = lane & 16, h3 = lane & 8, h2 = lane & 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = (h4 ? v[4 + i] : v[i]) + __shfl_xor_sync(0xffffffffu, h4 ? v[i] : v[4 + i], 16);
#pragma unroll
  for (int i = 0; i < 2; ++i) b[i] = (h3 ? a[2 + i] : a[i]) + __shfl_xor_sync(0xffffffffu, h3 ? a[i] : a[2 + i], 8);
  float c = (h2 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, h2 ? b[0] : b[1], 4);
  c += __shfl_xor_sync(0xffffffffu, c, 2);
  return c + __shfl_xor_sync(0xffffffffu, c, 1);
}

template <int BN, int TAIL, bool BY_K>
__global__ void __launch_bounds__(kThreads, 1)
linear_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_aux,
                   const __grid_constant__ CUtensorMap tm_out, const PairParams p) {
  using K = Cfg<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* tiles = ring + K::kStages * K::kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(tiles + 2 * K::kTile);      // in the leader: both CTAs' copies
  uint64_t* empty = full + K::kStages;
  uint64_t* acc_full = empty + K::kStages;           // [2]
  uint64_t* acc_empty = acc_full + 2;                // [2], in the leader: the group's warps in both CTAs
  uint64_t* ready = acc_empty + 2;                   // [2] the group's buffer: aux has come, or it is free
  uint64_t* done = ready + 2;                        // [2] the group's warps have written it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 2);

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
      ptx::mbar_init(&ready[i], 1);
      ptx::mbar_init(&done[i], kGroupWarps);
    }
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, 2 * BN);
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
          if (rank == 0) ptx::mbar_expect_tx(&full[st], 2 * K::kStage);
          const uint32_t bar = ptx::leader_addr(&full[st]);
          uint8_t *a = ring + st * K::kStage, *b = a + kBox;
          ptx::tma_load_4d_pair(a, &tm_a, bar, kb * 64, row0_of(i), 0, 0);
          if constexpr (BY_K) {
#pragma unroll
            for (int q = 0; q < BN / 128; ++q) ptx::tma_load_4d_pair(b + q * kRowsBox, &tm_b, bar, n0 + rank * (BN / 2) + q * 64, kb * 64, 0, 0);
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
      uint8_t* tile = tiles + g * K::kTile;
      for (int i = g; i < my_tiles; i += 2) {
        const int row0 = row0_of(i);
        if (TAIL != kPlainTail && p.has_aux) {
          ptx::mbar_expect_tx(&ready[g], K::kTile);
#pragma unroll
          for (int q = 0; q < BN / 64; ++q) ptx::tma_load_4d(tile + q * kBox, &tm_aux, &ready[g], n0 + q * 64, row0, 0, 0);
        } else {
          ptx::mbar_arrive(&ready[g]);
        }
        if (!ptx::mbar_wait(&done[g], i >> 1 & 1, 705)) break;
        if (row0 < p.rows) {
          for (int q = 0; q < BN / 64 && n0 + q * 64 < p.n; ++q) ptx::tma_store_4d(&tm_out, tile + q * kBox, n0 + q * 64, row0, 0, 0);
          ptx::tma_store_commit();
        }
        ptx::tma_store_wait_read();
      }
      ptx::tma_store_wait_all();
    }
  } else {
    // ---------------------------------------------------------------- the tail: a warp has 32 rows (tensor-memory lanes) of half of the columns
    const int g = (warp - kTailWarp) / kGroupWarps, quad = warp & 3, col0 = (warp - kTailWarp) / 4 % 2 * (BN / 2), r = quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + g * BN + col0;
    uint8_t* tile = tiles + g * K::kTile + r * 128;
    float sums[K::kChunks];                          // of column 8 (lane & 3) + what sum_rows gives, of each chunk
#pragma unroll
    for (int j = 0; j < K::kChunks; ++j) sums[j] = 0.f;
    for (int i = g; i < my_tiles; i += 2) {
      const uint32_t ph = i >> 1 & 1;
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&ready[g], ph, 706))) break;
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&acc_full[g], ph, 707))) break;
      ptx::tc_fence_after_sync();
#pragma unroll(TAIL == kBackwardTail ? K::kChunks : 1)
      for (int j = 0; j < K::kChunks; ++j) {
        uint32_t raw[32];
        ptx::tmem_ld_32x32b_x32(t_row + j * 32, raw);
        ptx::tmem_ld_wait();
        if (j + 1 == K::kChunks) {
          ptx::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(ptx::leader_addr(&acc_empty[g]));
        }
        const int col = col0 + j * 32;
        uint8_t* row = tile + col / 64 * kBox;
        auto cell_at = [&](int c) { return reinterpret_cast<uint4*>(row + (((col / 8 + c) & 7) ^ (r & 7)) * 16); };
        if constexpr (TAIL == kPlainTail) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = pack_bf16x2(__uint_as_float(raw[8 * c + 2 * q]), __uint_as_float(raw[8 * c + 2 * q + 1]));
            *cell_at(c) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          with_activation(p.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int at = n0 + col + 8 * c;
              float v[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) v[q] = __uint_as_float(raw[8 * c + q]);
              if (p.bias != nullptr && at < p.n) {          // (n is a multiple of 8)
                const float4 lo = *reinterpret_cast<const float4*>(p.bias + at), hi = *reinterpret_cast<const float4*>(p.bias + at + 4);
                v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w, v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
              }
              uint4* cell = cell_at(c);
              float x[8];
              if (TAIL == kBackwardTail || p.has_aux) {
                const uint4 a = *cell;
                const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int q = 0; q < 8; ++q) x[q] = __uint_as_float(q & 1 ? aw[q / 2] & 0xffff0000u : aw[q / 2] << 16);
              }
              if constexpr (TAIL == kForwardTail) {
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = activation<ACT>(v[q]);
                if (p.has_aux) {
#pragma unroll
                  for (int q = 0; q < 8; ++q) v[q] += x[q];
                }
              } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = x[q] * slope<ACT>(v[q]);
                if (p.partial != nullptr) {
                  const float s = sum_rows(v, lane);
                  if ((lane & 3) == c) sums[j] += s;
                }
              }
              uint32_t w[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) w[q] = pack_bf16x2(v[2 * q], v[2 * q + 1]);
              *cell = make_uint4(w[0], w[1], w[2], w[3]);
            }
          });
        }
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&done[g]);
    }
    if (TAIL == kBackwardTail && p.partial != nullptr) {
      // a row of partial sums for each pair of a column tile, group, CTA and quadrant
      float* row = p.partial + static_cast<long long>(((first * 2 + g) * 2 + rank) * 4 + quad) * p.n;
#pragma unroll
      for (int j = 0; j < K::kChunks; ++j) {
        const int at = n0 + col0 + j * 32 + 8 * (lane & 3) + 4 * (lane >> 4 & 1) + 2 * (lane >> 3 & 1) + (lane >> 2 & 1);
        if (at < p.n) row[at] = sums[j];
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncwarp();
  ptx::cluster_sync();      // neither CTA leaves while the other may still read its operands or reach its barriers
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem, 2 * BN);
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

// A tile's columns: 256, or 128 where these leave fewer of them unused.
int tile_width(int n) { return (n + 255) / 256 * 256 - n >= 128 ? 128 : 256; }

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

int backward_pairs(int n) { return tile_width(n) == 256 ? pairs_held<256, kBackwardTail, false>() : pairs_held<128, kBackwardTail, false>(); }

}  // namespace

bool linear_pair_ok(long long rows, int n, int k) {
  const int held = backward_pairs(n);
  if (held <= 0 || n < 64 || k < 64) return false;
  const Grid g = grid_of(rows, n, held);
  return g.groups > 0 && 4 * g.groups * g.n_tiles >= 3 * held;      // (three quarters of the pairs at least have a tile)
}

int linear_pair_partials(long long rows, int n, int k) { return grid_of(rows, n, backward_pairs(n)).groups * 16; }

int launch_linear_pair(cudaStream_t stream, const LinearPair& p, const char* tag) {
  KFB_CHECK_ARG((p.tail == kPlainTail) == (p.by_k != 0), "linear: tail %d with an operand %s k", p.tail, p.by_k ? "across" : "along");
  return tile_width(p.n) == 256 ? launch_width<256>(stream, p, tag) : launch_width<128>(stream, p, tag);
}

}  // namespace kfb
