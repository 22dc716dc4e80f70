// The gradients of the gated feed-forward's weights from x and dy alone, 128 channels, bf16:
//   a, b = x Wa^T, x Wb^T,  dh = dy Wo,  h = silu(a) b,  da = dh b silu'(a),  db = dh silu(a)
//   d[Wa; Wb] = [da, db]^T x,  dWo = dy^T h,  summed over a piece of the rows into a float32 plane.
//
// What bounds it.  The hidden channels are computed again: 6 products of rows x channels x hidden channels where the sums themselves are 3.  Kept from the
// kernel that has computed them for dx they would be 6 bytes per row and hidden channel to write, at the 4 TB/s that the memory takes (115 us for 147 456
// rows of 512 hidden channels), and as many to read.
//
// Split.  A CTA owns 64 hidden channels, their weights and their sums in tensor memory, and walks tiles of 128 rows; the CTAs that own other hidden
// channels walk the same rows, which come from L2 for all but one of them.
//   S   = [x [Wa; Wb]^T | dy Wo]      rows x 192
//   P   = da, db, h as bf16           in shared memory: sixteen warps, one S buffer
//   sums += x^T [da | db], dy^T h     channels x 192, every operand read across k as it lies: the tiles of x and dy serve both products
// One thread issues  S(i + 1), sums(i):  S runs under the element-wise part.  (With x^T and dy^T in tensor memory, 8 x 8 blocks transposed on their way by four
// more warps, the sums' products would be a third shorter; but the copy competes with S for shared memory, 1 500 cycles a tile, and the sums wait for it:
// 119 us where this is 106, 147 456 rows of 512 hidden channels.)  Bound by shared memory: 336 KB a tile, 2 600 cycles, and 2 990 for the products as they are.
#include <mutex>

#include "feed_forward_hidden.cuh"
#include "gemm.cuh"   // tanh_fast, pack_bf16x2, st_global_v8
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int C = 128, kRows = 128, kChunk = 64;
constexpr int kBox = kRows * 128;                    // [128 rows][64 bf16], 128-byte swizzle
constexpr int kSlot = 2 * kBox;                      // a tile of x, or of dy
constexpr int kWeights = 2 * kBox + kBox;            // [Wa; Wb] in two blocks of 64 k, Wo as it is stored
constexpr int kEpiWarp = 4, kEpiWarps = 16;          // four warps for each 32 rows, 16 hidden channels each
constexpr int kThreads = 32 * (kEpiWarp + kEpiWarps);
constexpr int kSmem = 4 * kSlot + kWeights + 3 * kBox + 512 + 1024;
static_assert(kSmem <= 232448, "shared memory");
constexpr uint32_t kSumAb = 0, kSumO = 128, kS = 192;     // tensor-memory columns

struct WeightsParams {
  int tiles, chunks, hidden, splits, units;
  float *dw_in, *dw_out;                             // planes (either may be null)
  long long plane_in, plane_out;
};

// Operands across k: rows of 128 bytes, one per k, eight of them (a swizzle atom) 1024 bytes apart, the next 64 elements a box further.
__device__ __forceinline__ uint64_t across_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(kBox >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

__global__ void __launch_bounds__(kThreads, 1)
ffn_weights_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_w1,
                   const __grid_constant__ CUtensorMap tm_wo, const WeightsParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* s_rows = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));   // x, dy, x, dy
  uint8_t* s_w = s_rows + 4 * kSlot;
  uint8_t* s_p = s_w + kWeights;                     // da, db, h
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_p + 3 * kBox);
  uint64_t* r_full = bars;                           // [4] in the order of the slots
  uint64_t* r_free = r_full + 4;
  uint64_t* w_full = r_free + 4;
  uint64_t* w_free = w_full + 1;
  uint64_t* s_full = w_free + 1;
  uint64_t* s_free = s_full + 1;
  uint64_t* p_full = s_free + 1;
  uint64_t* p_free = p_full + 1;
  uint64_t* o_full = p_free + 1;
  uint64_t* o_free = o_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto tiles_of = [&](int unit, int& t0) {           // of the unit's piece of the rows
    const int split = unit / p.chunks;
    t0 = static_cast<int>(static_cast<long long>(p.tiles) * split / p.splits);
    return static_cast<int>(static_cast<long long>(p.tiles) * (split + 1) / p.splits) - t0;
  };

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tm_x);
    ptx::prefetch_tmap(&tm_dy);
    for (int i = 0; i < 4; ++i) {
      ptx::mbar_init(&r_full[i], 1);
      ptx::mbar_init(&r_free[i], 1);
    }
    ptx::mbar_init(w_full, 1);
    ptx::mbar_init(w_free, 1);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(s_free, kEpiWarps);
    ptx::mbar_init(p_full, kEpiWarps);
    ptx::mbar_init(p_free, 1);
    ptx::mbar_init(o_full, 1);
    ptx::mbar_init(o_free, kEpiWarps);
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_enter();

  if (warp == 0) {
    // ---------------------------------------------------------------- rows and weights
    if (ptx::elect_one()) {
      bool ok = true;
      int round = 0;                                 // tiles so far
      uint32_t w_par = 1;
      for (int u = blockIdx.x; ok && u < p.units; u += gridDim.x, w_par ^= 1u) {
        int t0;
        const int n = tiles_of(u, t0), h0 = u % p.chunks * kChunk;
        ok = ptx::mbar_wait(w_free, w_par, 561);
        if (!ok) break;
        ptx::mbar_expect_tx(w_full, kWeights);
        for (int kb = 0; kb < 2; ++kb) {
          ptx::tma_load_4d(s_w + kb * kBox, &tm_w1, w_full, kb * 64, h0, 0, 0);
          ptx::tma_load_4d(s_w + kb * kBox + kBox / 2, &tm_w1, w_full, kb * 64, p.hidden + h0, 0, 0);
        }
        ptx::tma_load_4d(s_w + 2 * kBox, &tm_wo, w_full, h0, 0, 0, 0);
        for (int i = 0; ok && i < n; ++i, ++round) {
          for (int which = 0; which < 2; ++which) {
            const int slot = 2 * (round & 1) + which;
            const CUtensorMap* map = which ? &tm_dy : &tm_x;
            ok = ptx::mbar_wait(&r_free[slot], ((round >> 1) & 1) ^ 1, 562);
            if (!ok) break;
            ptx::mbar_expect_tx(&r_full[slot], kSlot);
            ptx::tma_load_4d(s_rows + slot * kSlot, map, &r_full[slot], 0, (t0 + i) * kRows, 0, 0);
            ptx::tma_load_4d(s_rows + slot * kSlot + kBox, map, &r_full[slot], 64, (t0 + i) * kRows, 0, 0);
          }
          // the tiles after the next two come into L2 meanwhile
          if (i + 2 < n) {
            for (int kb = 0; kb < 2; ++kb) {
              ptx::tma_prefetch_4d(&tm_x, kb * 64, (t0 + i + 2) * kRows, 0, 0);
              ptx::tma_prefetch_4d(&tm_dy, kb * 64, (t0 + i + 2) * kRows, 0, 0);
            }
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (ptx::elect_one()) {
      constexpr uint32_t kA = 1u << 15, kB = 1u << 16;        // operand across k
      constexpr uint32_t id_ab = ptx::make_idesc(kRows, 2 * kChunk, 1), id_dh = ptx::make_idesc(kRows, kChunk, 1) | kB;
      constexpr uint32_t id_dab = ptx::make_idesc(C, 2 * kChunk, 1) | kA | kB, id_dwo = ptx::make_idesc(C, kChunk, 1) | kA | kB;
      const uint64_t rows_k = ptx::make_kmajor_desc<128>(ptx::smem_u32(s_rows)), rows_x = across_desc(ptx::smem_u32(s_rows));
      const uint64_t w_ab = ptx::make_kmajor_desc<128>(ptx::smem_u32(s_w)), w_o = across_desc(ptx::smem_u32(s_w + 2 * kBox));
      const uint64_t p_ab = across_desc(ptx::smem_u32(s_p)), p_h = across_desc(ptx::smem_u32(s_p + 2 * kBox));
      bool ok = true;
      int round = 0, unit = 0;
      for (int u = blockIdx.x; ok && u < p.units; u += gridDim.x, ++unit) {
        int t0;
        const int n = tiles_of(u, t0);
        ok = ptx::mbar_wait(w_full, unit & 1, 563, ptx::kPolls);
        for (int i = -1; ok && i < n; ++i) {
          const int g = round + i;                            // tile i of this unit, and the next one's slots
          const int x1 = 2 * ((g + 1) & 1), x0 = 2 * (g & 1);
          if (i + 1 < n) {
            ok = ptx::mbar_wait(s_free, (g & 1), 564, ptx::kPolls) && ptx::mbar_wait(&r_full[x1], ((g + 1) >> 1) & 1, 565, ptx::kPolls);
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < 8; ++k)
              ptx::mma_f16_ss(tmem + kS, rows_k + x1 * (kSlot >> 4) + (k >> 2) * (kBox >> 4) + (k & 3) * 2, w_ab + (k >> 2) * (kBox >> 4) + (k & 3) * 2, id_ab,
                              k > 0 ? 1u : 0u);
          }
          if (i + 1 < n) {
            ok = ptx::mbar_wait(&r_full[x1 + 1], ((g + 1) >> 1) & 1, 568, ptx::kPolls);
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < 8; ++k)
              ptx::mma_f16_ss(tmem + kS + 128, rows_k + (x1 + 1) * (kSlot >> 4) + (k >> 2) * (kBox >> 4) + (k & 3) * 2, w_o + k * (2048 >> 4), id_dh,
                              k > 0 ? 1u : 0u);
            ptx::tc_commit(s_full);
            if (i + 2 == n) ptx::tc_commit(w_free);
          }
          if (i >= 0) {
            if (i == 0) ok = ptx::mbar_wait(o_free, (unit & 1) ^ 1, 566, ptx::kPolls);
            ok = ok && ptx::mbar_wait(p_full, g & 1, 567, ptx::kPolls);
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int k = 0; k < 8; ++k)
              ptx::mma_f16_ss(tmem + kSumAb, rows_x + x0 * (kSlot >> 4) + k * (2048 >> 4), p_ab + k * (2048 >> 4), id_dab, i > 0 || k > 0 ? 1u : 0u);
            ptx::tc_commit(&r_free[x0]);
          }
          if (i >= 0) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              ptx::mma_f16_ss(tmem + kSumO, rows_x + (x0 + 1) * (kSlot >> 4) + k * (2048 >> 4), p_h + k * (2048 >> 4), id_dwo, i > 0 || k > 0 ? 1u : 0u);
            ptx::tc_commit(&r_free[x0 + 1]);
            ptx::tc_commit(p_free);
          }
        }
        if (ok) ptx::tc_commit(o_full);
        round += n;
      }
    }
  } else if (warp >= kEpiWarp) {
    // ---------------------------------------------------------------- P, and the sums of a finished unit
    const int part = (warp - kEpiWarp) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    // 16-byte cells of a row's 128 bytes, swizzled: cell j of row r lies at j ^ (r % 8)
    uint8_t *cell0 = s_p + r * 128 + (((2 * part) ^ (r & 7)) << 4), *cell1 = s_p + r * 128 + (((2 * part + 1) ^ (r & 7)) << 4);
    bool ok = true;
    int round = 0, unit = 0;
    for (int u = blockIdx.x; ok && u < p.units; u += gridDim.x, ++unit) {
      int t0;
      const int n = tiles_of(u, t0);
      for (int i = 0; i < n; ++i, ++round) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(s_full, round & 1, 569)) != 0;
        if (!ok) break;
        ptx::tc_fence_after_sync();
        uint32_t a[16], b[16], g[16];
        ptx::tmem_ld_32x32b_x16(t_lane + kS + part * 16, a);
        ptx::tmem_ld_32x32b_x16(t_lane + kS + 64 + part * 16, b);
        ptx::tmem_ld_32x32b_x16(t_lane + kS + 128 + part * 16, g);
        ptx::tmem_ld_wait();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(s_free);
        uint32_t hw[8], aw[8], bw[8];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          // pairs: s = tanh(a / 2) / 2 + 1 / 2, silu = a s, silu' = s + silu (1 - s)
          const uint64_t half2 = ptx::pack2(0.5f, 0.5f), one2 = ptx::pack2(1.0f, 1.0f), minus2 = ptx::pack2(-1.0f, -1.0f);
          const uint64_t av = ptx::pack2(a[j], a[j + 1]), bv = ptx::pack2(b[j], b[j + 1]), gv = ptx::pack2(g[j], g[j + 1]);
          const float2 ah = ptx::unpack2(ptx::mul2(av, half2));
          const uint64_t sv = ptx::fma2(ptx::pack2(tanh_fast(ah.x), tanh_fast(ah.y)), half2, half2);
          const uint64_t silu = ptx::mul2(av, sv);
          const uint64_t slope = ptx::fma2(silu, ptx::fma2(sv, minus2, one2), sv);
          hw[j >> 1] = pack_bf16x2(ptx::mul2(silu, bv));
          aw[j >> 1] = pack_bf16x2(ptx::mul2(ptx::mul2(gv, bv), slope));
          bw[j >> 1] = pack_bf16x2(ptx::mul2(gv, silu));
        }
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(p_free, (round & 1) ^ 1, 570)) != 0;
        if (!ok) break;
        *reinterpret_cast<uint4*>(cell0) = make_uint4(aw[0], aw[1], aw[2], aw[3]);
        *reinterpret_cast<uint4*>(cell1) = make_uint4(aw[4], aw[5], aw[6], aw[7]);
        *reinterpret_cast<uint4*>(cell0 + kBox) = make_uint4(bw[0], bw[1], bw[2], bw[3]);
        *reinterpret_cast<uint4*>(cell1 + kBox) = make_uint4(bw[4], bw[5], bw[6], bw[7]);
        *reinterpret_cast<uint4*>(cell0 + 2 * kBox) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
        *reinterpret_cast<uint4*>(cell1 + 2 * kBox) = make_uint4(hw[4], hw[5], hw[6], hw[7]);
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_full);
      }
      if (!ok) break;
      // the unit's sums: lane = channel, column = hidden channel
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(o_full, unit & 1, 571)) != 0;
      if (!ok) break;
      ptx::tc_fence_after_sync();
      uint32_t ab[32], o[16];
      ptx::tmem_ld_32x32b_x32(t_lane + kSumAb + part * 32, ab);
      ptx::tmem_ld_32x32b_x16(t_lane + kSumO + part * 16, o);
      ptx::tmem_ld_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(o_free);
      const int split = u / p.chunks, h0 = u % p.chunks * kChunk;
      if (p.dw_in != nullptr) {
        float* d = p.dw_in + split * p.plane_in + static_cast<long long>((part >> 1) * p.hidden + h0 + (part & 1) * 32) * C + r;
#pragma unroll
        for (int j = 0; j < 32; ++j) d[j * C] = __uint_as_float(ab[j]);
      }
      if (p.dw_out != nullptr) {
        float* d = p.dw_out + split * p.plane_out + static_cast<long long>(r) * p.hidden + h0 + part * 16;
        st_global_v8(d, o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]);
        st_global_v8(d + 8, o[8], o[9], o[10], o[11], o[12], o[13], o[14], o[15]);
      }
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, 512);
  }
}

int matrix_map(CUtensorMap* m, const void* ptr, long long rows, long long cols, uint32_t box_rows) {
  const uint64_t dims[4] = {(uint64_t)cols, (uint64_t)rows, 1, 1};
  const uint64_t str[3] = {(uint64_t)cols * 2, (uint64_t)cols * 2 * rows, (uint64_t)cols * 2 * rows};
  const uint32_t box[4] = {64, box_rows, 1, 1};
  return make_tmap(m, ptr, 2, 4, dims, str, box, 128);
}

}  // namespace

bool ffn_weights_ok(int c, int hidden) { return c == C && hidden % kChunk == 0; }

int ffn_weights_planes(long long rows, int hidden) {
  const long long tiles = (rows + kRows - 1) / kRows, most = sm_count() / (hidden / kChunk);
  return static_cast<int>(most < 1 ? 1 : most < tiles ? most : tiles);
}

int launch_ffn_weights(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, float* dw_in, float* dw_out, int rows,
                       int hidden) {
  CUtensorMap tx, td, t1, to;
  KFB_TRY(matrix_map(&tx, x, rows, C, kRows));
  KFB_TRY(matrix_map(&td, dy, rows, C, kRows));
  KFB_TRY(matrix_map(&t1, w_in, 2ll * hidden, C, kChunk));
  KFB_TRY(matrix_map(&to, w_out, C, hidden, C));
  KFB_TRY(allow_smem<ffn_weights_kernel>(kSmem));
  WeightsParams p = {};
  p.tiles = cdiv(rows, kRows);
  p.chunks = hidden / kChunk;
  p.hidden = hidden;
  p.splits = ffn_weights_planes(rows, hidden);
  p.units = p.chunks * p.splits;
  p.dw_in = dw_in;
  p.dw_out = dw_out;
  p.plane_in = 2ll * hidden * C;
  p.plane_out = static_cast<long long>(hidden) * C;
  LaunchScope scope(stream, "feed_forward_weights_grad");
  return launch_kernel(stream, ffn_weights_kernel, p.units < sm_count() ? p.units : sm_count(), kThreads, kSmem, tx, td, t1, to, p);
}

}  // namespace kfb
