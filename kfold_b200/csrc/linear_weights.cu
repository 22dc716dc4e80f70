// The gradient of a linear layer's weights: plane[s][n][k] = sum over piece s of the rows of dz(r, n) x(r, k), bf16 operands, float32 planes.
//
// What bounds it: dz and x in, HBM, and their trips through shared memory.  A CTA pair (cta_group::2) multiplies 256 columns of dz by 256 of x over its piece
// of the rows, so that each operand is read by few pairs; all operands lie across the contraction and are read as they lie.  The bias's gradient, where dz is the
// gradient itself, is one more product with columns of ones: a pass over dz and a launch less.
// 147 456 rows, 512 x 256: 44 us (0.87 PFLOP/s, 5.1 TB/s) and 8 for the planes; 18 432 rows, 384 x 1 536: 25 us (0.87 PFLOP/s) and 6.
#include <mutex>

#include "gemm.cuh"   // st_global_v8
#include "linear_tail.cuh"
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int kK = 64;                               // rows of a block
constexpr int kBox = kK * 128;                       // [64 rows][64 columns], 128-byte swizzle
constexpr int kOperand = 2 * kBox, kStage = 2 * kOperand, kStages = 6;      // 128 columns of each operand
constexpr int kTile = 256;
constexpr int kTailWarp = 4, kTailWarps = 8;
constexpr int kThreads = 32 * (kTailWarp + kTailWarps);
constexpr int kOnes = 4096;                          // bytes of ones: the operand whose product with dz is its sums over rows, whatever its layout
constexpr int kOnesColumns = 32;                     // of the pair
constexpr int kSmem = kStages * kStage + kOnes + 512 + 1024;

struct WeightParams {
  int n, k, blocks, splits, n_tiles, tiles, add;     // blocks of 64 rows
  float *planes, *bias_planes;
};

__device__ __forceinline__ uint64_t across_desc(uint32_t addr) {   // rows of 128 bytes, one per row of the operand; the next 64 columns a box further
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(kBox >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__global__ void __launch_bounds__(kThreads, 1)
linear_weights_kernel(const __grid_constant__ CUtensorMap tm_dz, const __grid_constant__ CUtensorMap tm_x, const WeightParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ones = ring + kStages * kStage;
  uint64_t* full = reinterpret_cast<uint64_t*>(ones + kOnes);                // in the leader: both CTAs' copies
  uint64_t* empty = full + kStages;
  uint64_t* done = empty + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int unit = blockIdx.x >> 1, tile = unit % p.tiles, split = unit / p.tiles;
  const int n0 = tile % p.n_tiles * kTile + rank * 128, k0 = tile / p.n_tiles * kTile;      // dz's columns of this CTA, x's of the pair
  const int b0 = static_cast<int>(static_cast<long long>(p.blocks) * split / p.splits);
  const int b1 = static_cast<int>(static_cast<long long>(p.blocks) * (split + 1) / p.splits);

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tm_dz);
    ptx::prefetch_tmap(&tm_x);
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], 1);
    }
    ptx::mbar_init(done, 1);
    ptx::fence_barrier_init();
  }
  // (the tiles that share these columns of dz share this work: a block of rows is one's)
  const bool bias = p.bias_planes != nullptr;
  const int k_tiles = p.tiles / p.n_tiles, turn = tile / p.n_tiles;
  int first_bias = b0 + (turn - b0 % k_tiles + k_tiles) % k_tiles;      // the first block of this tile's
  for (int i = threadIdx.x; i < kOnes / 4; i += kThreads) reinterpret_cast<uint32_t*>(ones)[i] = 0x3f803f80u;
  ptx::fence_proxy_async_smem();
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, 512);
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
      for (int b = b0; b < b1; ++b) {
        ok = ptx::mbar_wait(&empty[st], ph ^ 1, 721);
        if (!ok) break;
        if (rank == 0) ptx::mbar_expect_tx(&full[st], 2 * kStage);
        const uint32_t bar = ptx::leader_addr(&full[st]);
        uint8_t* s = ring + st * kStage;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          ptx::tma_load_4d_pair(s + q * kBox, &tm_dz, bar, n0 + q * 64, b * kK, 0, 0);
          ptx::tma_load_4d_pair(s + kOperand + q * kBox, &tm_x, bar, k0 + rank * 128 + q * 64, b * kK, 0, 0);
        }
        if (++st == kStages) { st = 0; ph ^= 1u; }
      }
      for (int i = 0; ok && i < kStages; ++i) {     // the last products' arrivals at this CTA's barriers, before it may exit
        ok = ptx::mbar_wait(&empty[st], ph ^ 1, 722);
        if (++st == kStages) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && ptx::elect_one()) {
      constexpr uint32_t idesc = ptx::make_idesc(256, kTile, 1) | (1u << 15) | (1u << 16);
      constexpr uint32_t ones_idesc = ptx::make_idesc(256, kOnesColumns, 1) | (1u << 15);
      const uint64_t d0 = across_desc(ptx::smem_u32(ring)), ones_desc = ptx::make_kmajor_desc<128>(ptx::smem_u32(ones));
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int b = b0; b < b1; ++b) {
        ok = ptx::mbar_wait(&full[st], ph, 723, ptx::kPolls);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint64_t a = d0 + st * (kStage >> 4), x = a + (kOperand >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) ptx::mma_f16_ss_pair(tmem, a + k * (2048 >> 4), x + k * (2048 >> 4), idesc, b > b0 || k > 0 ? 1u : 0u);
        if (bias && b % k_tiles == turn) {
#pragma unroll
          for (int k = 0; k < 4; ++k) ptx::mma_f16_ss_pair(tmem + kTile, a + k * (2048 >> 4), ones_desc, ones_idesc, b > first_bias || k > 0 ? 1u : 0u);
        }
        ptx::tc_commit_pair(&empty[st]);
        if (++st == kStages) { st = 0; ph ^= 1u; }
      }
      if (ok) ptx::tc_commit_pair(done);
    }
  } else if (warp >= kTailWarp) {
    // lane = column of dz, tensor-memory column = column of x; a warp takes half of these
    const int quad = warp & 3, n = n0 + quad * 32 + lane, c0 = (warp - kTailWarp) / 4 * (kTile / 2);
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const bool ok = __all_sync(0xffffffffu, ptx::mbar_wait(done, 0, 724)) != 0;
    ptx::tc_fence_after_sync();
    if (ok) {
      if (bias && c0 == 0) {
        uint32_t v[8];
        ptx::tmem_ld_32x32b_x8(t_row + kTile, v);
        ptx::tmem_ld_wait();
        if (n < p.n) {
          float* d = p.bias_planes + (static_cast<long long>(split) * k_tiles + turn) * p.n + n;
          *d = first_bias < b1 ? __uint_as_float(v[0]) : 0.f;
        }
      }
      float* d = p.planes + (static_cast<long long>(split) * p.n + n) * p.k + k0;
#pragma unroll 1
      for (int c = c0; c < c0 + kTile / 2; c += 32) {
        uint32_t v[32];
        __syncwarp();
        ptx::tmem_ld_32x32b_x32(t_row + c, v);
        ptx::tmem_ld_wait();
        if (n >= p.n) continue;
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (k0 + c + j >= p.k) continue;           // (k is a multiple of 8)
          if (p.add) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j + i] = __float_as_uint(__uint_as_float(v[j + i]) + d[c + j + i]);
          }
          st_global_v8(d + c + j, v[j], v[j + 1], v[j + 2], v[j + 3], v[j + 4], v[j + 5], v[j + 6], v[j + 7]);
        }
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncwarp();
  ptx::cluster_sync();      // neither CTA leaves while the other may still read its operands or reach its barriers
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem, 512);
  }
}

int pairs_held() {
  static std::once_flag once[64];
  static int held[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::call_once(once[dev & 63], [&] { held[dev & 63] = clusters_held(linear_weights_kernel, 2, kThreads, kSmem); });
  return held[dev & 63];
}

int matrix_map(CUtensorMap* m, const void* ptr, long long rows, long long cols) {
  const uint64_t dims[4] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows), 1, 1};
  const uint64_t str[3] = {static_cast<uint64_t>(cols) * 2, static_cast<uint64_t>(cols) * 2 * rows, static_cast<uint64_t>(cols) * 2 * rows};
  const uint32_t box[4] = {64, kK, 1, 1};
  return make_tmap(m, ptr, 2, 4, dims, str, box, 128);
}
int tiles_of(int n, int k) { return cdiv(n, kTile) * cdiv(k, kTile); }

}  // namespace

// Many rows: a pair's start and end, and the planes of all pairs, cost more than tiles of 128 x 128 do (matmul.cu) until the products take some microseconds, half
// as many where a pass over dz for the bias's gradient goes with it.  By pairs and by tiles, bf16: 768 x 768, 4 096 rows 24 and 24 us, 24 576 rows 34 and 40;
// 512 x 256, 8 192 rows 19 and 12, 49 152 rows 30 and 30; with the bias's gradient 19 and 17, 30 and 38;
// 63 001 rows of 128 x 128 (half of a tile unused) 15 and 13.
bool linear_weights_ok(long long rows, int n, int k, bool with_bias) {
  const double products = static_cast<double>(rows) * n * k;
  return rows >= 4096 && n >= 256 && k >= 256 && products >= (with_bias ? 2.5e9 : 5e9) && tiles_of(n, k) <= pairs_held();
}

int linear_weights_bias_planes(int splits, int k) { return splits * cdiv(k, kTile); }

int linear_weights_splits(long long rows, int n, int k) {
  const long long blocks = (rows + kK - 1) / kK, most = pairs_held() / tiles_of(n, k);
  return static_cast<int>(most < 1 ? 1 : most < blocks ? most : blocks);
}

int launch_linear_weights(cudaStream_t stream, const void* dz, const void* x, float* planes, float* bias_planes, int splits, int add, long long rows, int n,
                          int k) {
  CUtensorMap ta, tb;
  KFB_TRY(matrix_map(&ta, dz, rows, n));
  KFB_TRY(matrix_map(&tb, x, rows, k));
  KFB_CHECK_ARG(pairs_held() > 0, "linear: the device holds no pair of this kernel");
  KFB_CHECK_ARG(bias_planes == nullptr || !add, "linear: sums of dz over one piece of the rows only");
  WeightParams p = {};
  p.n = n;
  p.k = k;
  p.blocks = static_cast<int>((rows + kK - 1) / kK);
  p.splits = splits < p.blocks ? splits : p.blocks;
  p.n_tiles = cdiv(n, kTile);
  p.tiles = tiles_of(n, k);
  p.add = add;
  p.planes = planes;
  p.bias_planes = bias_planes;
  LaunchScope scope(stream, "linear_weights");
  return launch_kernel_clustered(stream, linear_weights_kernel, 2, 2 * p.tiles * p.splits, kThreads, kSmem, ta, tb, p);
}

}  // namespace kfb
