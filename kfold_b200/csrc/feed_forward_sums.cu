// The gradients of the gated feed-forward's weights from the hidden channels' that are kept, 256 channels, bf16:
//   d[Wa; Wb] = [da, db]^T x,  dWo = dy^T h,  summed over a piece of the rows into a float32 plane.
//
// What bounds it: 6 bytes per row and hidden channel to read, and the products of what was read with 256 channels, about as long either way.  Every operand
// is read once if a tile has all channels: a CTA pair multiplies 512 hidden columns, two products of 256 x 256 that share the block of x (or dy), each CTA
// half of the columns and half of the channels.  (Products of 128 columns by 128 channels, each operand from shared memory, spend two fifths of their time
// on reading the left one: 163 cycles for 256 x 16 values of it where its products are 128, 103 for 64.)  All operands lie across the contraction and are
// read as they lie.
// Measured: 147 456 rows of 1 024 hidden channels 177 us (141 at the measured burst rate; 905 MB take 138); 217 by products of 128 x 128.
#include <mutex>

#include "feed_forward_hidden.cuh"
#include "gemm.cuh"   // st_global_v8
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int C = 256, kK = 64;                      // rows of a block
constexpr int kBox = kK * 128;                       // [64 rows][64 columns], 128-byte swizzle
constexpr int kAPart = 2 * kBox, kStage = 2 * kAPart + 2 * kBox, kStages = 4;   // 2 x 128 columns, 128 channels
constexpr int kColumns = 512;                        // of a pair
constexpr int kEpiWarp = 4, kEpiWarps = 8;
constexpr int kThreads = 32 * (kEpiWarp + kEpiWarps);
constexpr int kSmem = kStages * kStage + 512 + 1024;

struct SumsParams {
  int hidden, blocks, splits, tiles_in, tiles;       // blocks of 64 rows; column tiles of [da, db], and with those of h
  int add;                                           // to what the planes hold
  float *dw_in, *dw_out;                             // planes
  long long plane_in, plane_out;
};

__device__ __forceinline__ uint64_t across_desc(uint32_t addr) {   // rows of 128 bytes, one per k; the next 64 columns a box further
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(kBox >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__global__ void __launch_bounds__(kThreads, 1)
ffn_sums_pair_kernel(const __grid_constant__ CUtensorMap tm_dab, const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_h,
                     const __grid_constant__ CUtensorMap tm_dy, const SumsParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * kStage);     // in the leader: both CTAs' copies
  uint64_t* empty = full + kStages;
  uint64_t* done = empty + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int unit = blockIdx.x >> 1, tile = unit % p.tiles, split = unit / p.tiles;
  const bool out = tile >= p.tiles_in;                                       // of h and dy
  const int g0 = (out ? tile - p.tiles_in : tile) * kColumns + rank * 128;   // this CTA's first column, and 256 on
  const int b0 = static_cast<int>(static_cast<long long>(p.blocks) * split / p.splits);
  const int b1 = static_cast<int>(static_cast<long long>(p.blocks) * (split + 1) / p.splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], 1);
    }
    ptx::mbar_init(done, 1);
    ptx::fence_barrier_init();
  }
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
      const CUtensorMap *ma = out ? &tm_h : &tm_dab, *mb = out ? &tm_dy : &tm_x;
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int b = b0; b < b1; ++b) {
        ok = ptx::mbar_wait(&empty[st], ph ^ 1, 581);
        if (!ok) break;
        if (rank == 0) ptx::mbar_expect_tx(&full[st], 2 * kStage);
        const uint32_t bar = ptx::leader_addr(&full[st]);
        uint8_t* s = ring + st * kStage;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q) ptx::tma_load_4d_pair(s + t * kAPart + q * kBox, ma, bar, g0 + t * 256 + q * 64, b * kK, 0, 0);
#pragma unroll
        for (int q = 0; q < 2; ++q) ptx::tma_load_4d_pair(s + 2 * kAPart + q * kBox, mb, bar, rank * 128 + q * 64, b * kK, 0, 0);
        if (++st == kStages) { st = 0; ph ^= 1u; }
      }
      for (int i = 0; ok && i < kStages; ++i) {     // the last products' arrivals at this CTA's barriers, before it may exit
        ok = ptx::mbar_wait(&empty[st], ph ^ 1, 582);
        if (++st == kStages) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && ptx::elect_one()) {
      constexpr uint32_t idesc = ptx::make_idesc(256, C, 1) | (1u << 15) | (1u << 16);
      const uint64_t d0 = across_desc(ptx::smem_u32(ring));
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int b = b0; b < b1; ++b) {
        ok = ptx::mbar_wait(&full[st], ph, 583, ptx::kPolls);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint64_t a = d0 + st * (kStage >> 4), bd = a + (2 * kAPart >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            ptx::mma_f16_ss_pair(tmem + t * C, a + t * (kAPart >> 4) + k * (2048 >> 4), bd + k * (2048 >> 4), idesc, b > b0 || k > 0 ? 1u : 0u);
        ptx::tc_commit_pair(&empty[st]);
        if (++st == kStages) { st = 0; ph ^= 1u; }
      }
      if (ok) ptx::tc_commit_pair(done);
    }
  } else if (warp >= kEpiWarp) {
    // lane = hidden column, tensor-memory column = channel; a warp takes one of the two products
    const int t = (warp - kEpiWarp) >> 2, quad = warp & 3, g = g0 + t * 256 + quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + t * C;
    const bool ok = __all_sync(0xffffffffu, ptx::mbar_wait(done, 0, 584)) != 0;
    ptx::tc_fence_after_sync();
    if (ok) {
      const bool mine = g < (out ? p.hidden : 2 * p.hidden);
      float* d = out ? p.dw_out + split * p.plane_out + g : p.dw_in + split * p.plane_in + static_cast<long long>(g) * C;
#pragma unroll 1
      for (int c = 0; c < C; c += 32) {
        uint32_t v[32];
        ptx::tmem_ld_32x32b_x32(t_row + c, v);
        ptx::tmem_ld_wait();
        if (!mine) continue;
        if (p.add) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) + d[out ? static_cast<long long>(c + j) * p.hidden : c + j]);
        }
        if (out) {
#pragma unroll
          for (int j = 0; j < 32; ++j) d[static_cast<long long>(c + j) * p.hidden] = __uint_as_float(v[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 8) st_global_v8(d + c + j, v[j], v[j + 1], v[j + 2], v[j + 3], v[j + 4], v[j + 5], v[j + 6], v[j + 7]);
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
  std::call_once(once[dev & 63], [&] { held[dev & 63] = clusters_held(ffn_sums_pair_kernel, 2, kThreads, kSmem); });
  return held[dev & 63];
}

int matrix_map(CUtensorMap* m, const void* ptr, long long rows, long long cols) {
  const uint64_t dims[4] = {(uint64_t)cols, (uint64_t)rows, 1, 1};
  const uint64_t str[3] = {(uint64_t)cols * 2, (uint64_t)cols * 2 * rows, (uint64_t)cols * 2 * rows};
  const uint32_t box[4] = {64, kK, 1, 1};
  return make_tmap(m, ptr, 2, 4, dims, str, box, 128);
}

}  // namespace

bool ffn_sums_ok(int c, int hidden) { return c == C && hidden % 64 == 0 && pairs_held() > 0; }

int ffn_sums_planes(long long rows, int hidden) {
  const int tiles = cdiv(2 * hidden, kColumns) + cdiv(hidden, kColumns), held = pairs_held();
  const long long blocks = (rows + kK - 1) / kK, most = held / tiles;
  return static_cast<int>(most < 1 ? 1 : most < blocks ? most : blocks);
}

int launch_ffn_sums(cudaStream_t stream, const void* dab, const void* x, const void* h, const void* dy, float* dw_in, float* dw_out, int splits, int add,
                    int rows, int hidden) {
  CUtensorMap ta, tx, th, td;
  KFB_TRY(matrix_map(&ta, dab, rows, 2ll * hidden));
  KFB_TRY(matrix_map(&tx, x, rows, C));
  KFB_TRY(matrix_map(&th, h, rows, hidden));
  KFB_TRY(matrix_map(&td, dy, rows, C));
  KFB_CHECK_ARG(pairs_held() > 0, "feed_forward: the device holds no pair of this kernel");
  SumsParams p = {};
  p.hidden = hidden;
  p.blocks = cdiv(rows, kK);
  p.splits = splits < p.blocks ? splits : p.blocks;
  p.tiles_in = dw_in != nullptr ? cdiv(2 * hidden, kColumns) : 0;
  p.tiles = p.tiles_in + (dw_out != nullptr ? cdiv(hidden, kColumns) : 0);
  p.add = add;
  p.dw_in = dw_in;
  p.dw_out = dw_out;
  p.plane_in = 2ll * hidden * C;
  p.plane_out = static_cast<long long>(hidden) * C;
  LaunchScope scope(stream, "feed_forward_sums");
  return launch_kernel_clustered(stream, ffn_sums_pair_kernel, 2, 2 * p.tiles * p.splits, kThreads, kSmem, ta, tx, th, td, p);
}

}  // namespace kfb
