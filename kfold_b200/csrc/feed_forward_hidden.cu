// Hidden channels of the gated feed-forward and their gradients:  a, b = x Wa^T, x Wb^T,  dh = dy Wo,
//   h = silu(a) b,   da = dh b silu'(a),   db = dh silu(a)
// as one kernel: three products into tensor memory, the element-wise part on the way out, h, da and db written once in bf16 (the operands of the
// gradients' products).  a, b and dh stay float32 and are never stored.
//
// sigmoid(a) = tanh(a / 2) / 2 + 1 / 2 by tanh.approx, one operation of the special function unit where an exponential and a reciprocal are two; all bf16 kernels of the
// feed-forward take it so.  What that costs, y, dx and the weights' gradients against 64 bits, every gate near one value: 2.3e-3 of their root mean square
// from 8 down to -4 (the rounding of h, da and db), 2.7e-3 near -8, 4.6e-3 near -10, 5.9e-3 near -12 (torch's bf16 operations: 3.9e-3 near 0, 1e-2 near -8, 1.6e-2
// near -10).  Below, the sum with 1 / 2 has no bits left for a sigmoid under 2^-20: 2e-2 near -14, and nothing of a result of 1e-7 near -16, where
// the float32-accurate mode keeps it.
//
// Split.  A CTA pair takes 256 rows, 128 in each CTA, and walks hidden channels in chunks of 64: [a | b] is one product of 128 columns (CTA 0 loads
// the chunk's rows of Wa, CTA 1 those of Wb), dh one of 64 with Wo read as it is stored, across k.  Up to 256 channels the rows of x and dy stay in
// shared memory for all chunks of a tile and only weights stream, 12 KB a CTA per 416 cycles of products; wider rows stream too.
// Two S buffers of 192 columns: sixteen warps take a chunk's element-wise part while the next is multiplied.  (Eight in two groups that took the
// chunks in turn, 32 channels at a time, waited out every latency: 3 960 cycles a chunk where its products are 1 664.)
// What bounds it: at 128 channels the 6 bytes per row and hidden channel that it writes, at 256 that and the products alike.  147 456 rows of 512 hidden
// channels, for the gradient: 107 us, 453 MB at 4.2 TB/s (writes alone reach 4), 64 without its stores.  Of 128 and 256 channels with many rows the
// kernels that have dx too take its place; few rows: a unit is fewer chunks, so that they fill the device (331 rows of 384 channels: 10 us).
#include "feed_forward_hidden.cuh"

#include <mutex>

#include "gemm.cuh"   // tanh_fast, pack_bf16x2
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int kRows = 128, kChunk = 64;
constexpr int kBox = kRows * 128;                    // [128 rows][64 bf16], 128-byte swizzle
constexpr int kRowSlot = 2 * kBox, kRowSlots = 4;    // a 64-wide block of x and of dy
constexpr int kW1 = 64 * 128, kWo = 64 * 64;         // a CTA's [64 hidden][64 k] of Wa or Wb, and [64 k][32 hidden] of Wo (64-byte swizzle)
constexpr int kWSlot = kW1 + kWo, kWSlots = 8;
constexpr int kEpiWarp = 4, kEpiWarps = 16;          // four warps for each 32 rows, 16 hidden channels each
constexpr int kThreads = 32 * (kEpiWarp + kEpiWarps);
constexpr int kS = 192;                              // tensor-memory columns of an S buffer
constexpr int kSmem = kRowSlots * kRowSlot + kWSlots * kWSlot + 512 + 1024;
static_assert(kSmem <= 232448, "shared memory");

struct HiddenParams {
  int rows, k_blocks, chunks, hidden;
  int groups, per_group, units;                      // a unit: a row block and `per_group` chunks
  int resident;                                      // the rows of a unit stay in shared memory
  __nv_bfloat16 *h, *dab;                            // 32-byte aligned, as their rows are
};

__device__ __forceinline__ uint64_t wo_desc(uint32_t addr) {   // [k][32 hidden] rows of 64 bytes, eight of them (a swizzle atom) 512 bytes apart
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (1ull << 16) | (static_cast<uint64_t>(512 >> 4) << 32) | (1ull << 46) | (4ull << 61);
}

template <bool GRAD>
__global__ void __launch_bounds__(kThreads, 1)
ffn_hidden_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_w1,
                       const __grid_constant__ CUtensorMap tm_wo, const HiddenParams p) {
  constexpr int kRowBytes = GRAD ? kRowSlot : kBox, kWBytes = GRAD ? kWSlot : kW1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* s_rows = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_w = s_rows + kRowSlots * kRowSlot;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_w + kWSlots * kWSlot);
  uint64_t* w_full = bars;                        // in the leader: both CTAs' copies
  uint64_t* w_free = w_full + kWSlots;
  uint64_t* r_full = w_free + kWSlots;            // in the leader
  uint64_t* r_free = r_full + kRowSlots;
  uint64_t* s_full = r_free + kRowSlots;          // [2]
  uint64_t* s_free = s_full + 2;                  // [2], in the leader: the element-wise warps of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int unit0 = blockIdx.x >> 1, unit_step = gridDim.x >> 1;
  auto chunks_of = [&](int unit, int& c0) {
    c0 = unit % p.groups * p.per_group;
    return min(p.per_group, p.chunks - c0);
  };
  auto row0_of = [&](int unit) { return (2 * (unit / p.groups) + rank) * kRows; };

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tm_x);
    ptx::prefetch_tmap(&tm_w1);
    for (int i = 0; i < kWSlots; ++i) {
      ptx::mbar_init(&w_full[i], 1);
      ptx::mbar_init(&w_free[i], 1);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      ptx::mbar_init(&r_full[i], 1);
      ptx::mbar_init(&r_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&s_free[i], 2 * kEpiWarps);
    }
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
    // ---------------------------------------------------------------- weights
    if (ptx::elect_one()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = unit0; ok && u < p.units; u += unit_step) {
        int c0;
        const int n = chunks_of(u, c0);
        for (int c = c0; ok && c < c0 + n; ++c)
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            ok = ptx::mbar_wait(&w_free[st], ph ^ 1, 521);
            if (!ok) break;
            if (rank == 0) ptx::mbar_expect_tx(&w_full[st], 2 * kWBytes);
            const uint32_t bar = ptx::leader_addr(&w_full[st]);
            ptx::tma_load_4d_pair(s_w + st * kWSlot, &tm_w1, bar, kb * 64, rank * p.hidden + c * kChunk, 0, 0);
            if (GRAD) ptx::tma_load_4d_pair(s_w + st * kWSlot + kW1, &tm_wo, bar, c * kChunk + rank * 32, kb * 64, 0, 0);
            if (++st == kWSlots) { st = 0; ph ^= 1u; }
          }
      }
      for (int i = 0; ok && i < kWSlots; ++i) {     // the last products' arrivals at this CTA's barriers, before it may exit
        ok = ptx::mbar_wait(&w_free[st], ph ^ 1, 522);
        if (++st == kWSlots) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- rows
    if (ptx::elect_one()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int u = unit0; ok && u < p.units; u += unit_step) {
        int c0;
        const int rounds = p.resident ? 1 : chunks_of(u, c0);
        // (where a unit fills all slots, the next one's rows come at once when they fall free: from L2)
        if (p.resident && u + unit_step < p.units)
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            ptx::tma_prefetch_4d(&tm_x, kb * 64, row0_of(u + unit_step), 0, 0);
            if (GRAD) ptx::tma_prefetch_4d(&tm_dy, kb * 64, row0_of(u + unit_step), 0, 0);
          }
        for (int c = 0; ok && c < rounds; ++c)
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            ok = ptx::mbar_wait(&r_free[st], ph ^ 1, 523);
            if (!ok) break;
            if (rank == 0) ptx::mbar_expect_tx(&r_full[st], 2 * kRowBytes);
            const uint32_t bar = ptx::leader_addr(&r_full[st]);
            ptx::tma_load_4d_pair(s_rows + st * kRowSlot, &tm_x, bar, kb * 64, row0_of(u), 0, 0);
            if (GRAD) ptx::tma_load_4d_pair(s_rows + st * kRowSlot + kBox, &tm_dy, bar, kb * 64, row0_of(u), 0, 0);
            if (++st == kRowSlots) { st = 0; ph ^= 1u; }
          }
      }
      for (int i = 0; ok && i < kRowSlots; ++i) {
        ok = ptx::mbar_wait(&r_free[st], ph ^ 1, 524);
        if (++st == kRowSlots) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (rank == 0 && ptx::elect_one()) {
      constexpr uint32_t idesc_s = ptx::make_idesc(2 * kRows, 2 * kChunk, 1), idesc_g = ptx::make_idesc(2 * kRows, kChunk, 1) | (1u << 16);
      const uint64_t row_desc = ptx::make_kmajor_desc<128>(ptx::smem_u32(s_rows));
      const uint64_t w1_desc = ptx::make_kmajor_desc<128>(ptx::smem_u32(s_w)), g_desc = wo_desc(ptx::smem_u32(s_w) + kW1);
      int st = 0, rs = 0, s = 0;
      uint32_t ph = 0, r_ph = 0, s_ph = 1;
      bool ok = true;
      for (int u = unit0; ok && u < p.units; u += unit_step) {
        int c0;
        const int n = chunks_of(u, c0);
        const int rs0 = rs;
        const uint32_t r_ph0 = r_ph;
        for (int c = 0; ok && c < n; ++c) {
          ok = ptx::mbar_wait(&s_free[s], s_ph, 525, ptx::kPolls);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const uint32_t d = tmem + s * kS;
          if (p.resident) { rs = rs0; r_ph = r_ph0; }
          const bool fresh_rows = !p.resident || c == 0, last_rows = !p.resident || c == n - 1;
          for (int kb = 0; kb < p.k_blocks; ++kb) {
            if (fresh_rows) ok = ptx::mbar_wait(&r_full[rs], r_ph, 526, ptx::kPolls);
            ok = ok && ptx::mbar_wait(&w_full[st], ph, 527, ptx::kPolls);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const uint64_t xd = row_desc + rs * (kRowSlot >> 4), wd = w1_desc + st * (kWSlot >> 4), gd = g_desc + st * (kWSlot >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) ptx::mma_f16_ss_pair(d, xd + k * 2, wd + k * 2, idesc_s, kb > 0 || k > 0 ? 1u : 0u);
            if (GRAD) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                ptx::mma_f16_ss_pair(d + 128, xd + (kBox >> 4) + k * 2, gd + k * (1024 >> 4), idesc_g, kb > 0 || k > 0 ? 1u : 0u);
            }
            ptx::tc_commit_pair(&w_free[st]);
            if (last_rows) ptx::tc_commit_pair(&r_free[rs]);
            if (++st == kWSlots) { st = 0; ph ^= 1u; }
            if (++rs == kRowSlots) { rs = 0; r_ph ^= 1u; }
          }
          if (!ok) break;
          ptx::tc_commit_pair(&s_full[s]);
          s ^= 1;
          if (s == 0) s_ph ^= 1u;
        }
      }
    }
  } else if (warp >= kEpiWarp) {
    // ---------------------------------------------------------------- h, da, db
    const int part = (warp - kEpiWarp) >> 2, quad = warp & 3;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16) + part * 16;
    int s = 0;
    uint32_t par = 0;
    bool ok = true;
    for (int u = unit0; ok && u < p.units; u += unit_step) {
      int c0;
      const int n = chunks_of(u, c0), row = row0_of(u) + quad * 32 + lane;
      __nv_bfloat16 *h_row = p.h + static_cast<long long>(row) * p.hidden + part * 16, *g_row = p.dab + 2ll * row * p.hidden + part * 16;
      for (int c = c0; c < c0 + n; ++c) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&s_full[s], par, 528)) != 0;
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t t = t_row + s * kS;
        uint32_t a[16], b[16], g[16];
        ptx::tmem_ld_32x32b_x16(t, a);
        ptx::tmem_ld_32x32b_x16(t + 64, b);
        if (GRAD) ptx::tmem_ld_32x32b_x16(t + 128, g);
        ptx::tmem_ld_wait();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_cluster(ptx::leader_addr(&s_free[s]));
        s ^= 1;
        if (s == 0) par ^= 1u;
        uint32_t hw[8], aw[8], bw[8];
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          // pairs: s = tanh(a / 2) / 2 + 1 / 2, silu = a s, silu' = s + silu (1 - s)
          const uint64_t half2 = ptx::pack2(0.5f, 0.5f), one2 = ptx::pack2(1.0f, 1.0f), minus2 = ptx::pack2(-1.0f, -1.0f);
          const uint64_t av = ptx::pack2(a[j], a[j + 1]), bv = ptx::pack2(b[j], b[j + 1]);
          const float2 ah = ptx::unpack2(ptx::mul2(av, half2));
          const uint64_t sv = ptx::fma2(ptx::pack2(tanh_fast(ah.x), tanh_fast(ah.y)), half2, half2);
          const uint64_t silu = ptx::mul2(av, sv);
          hw[j >> 1] = pack_bf16x2(ptx::mul2(silu, bv));
          if (GRAD) {
            const uint64_t gv = ptx::pack2(g[j], g[j + 1]);
            const uint64_t slope = ptx::fma2(silu, ptx::fma2(sv, minus2, one2), sv);
            aw[j >> 1] = pack_bf16x2(ptx::mul2(ptx::mul2(gv, bv), slope));
            bw[j >> 1] = pack_bf16x2(ptx::mul2(gv, silu));
          }
        }
        // a whole 32-byte sector of each array a thread; the four warps of these rows fill their lines together
        if (row < p.rows) {
          const int at = c * kChunk;
          st_global_v8(h_row + at, hw[0], hw[1], hw[2], hw[3], hw[4], hw[5], hw[6], hw[7]);
          if (GRAD) {
            st_global_v8(g_row + at, aw[0], aw[1], aw[2], aw[3], aw[4], aw[5], aw[6], aw[7]);
            st_global_v8(g_row + p.hidden + at, bw[0], bw[1], bw[2], bw[3], bw[4], bw[5], bw[6], bw[7]);
          }
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

template <bool GRAD>
int pairs_held() {
  static std::once_flag once[64];
  static int held[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::call_once(once[dev & 63], [&] { held[dev & 63] = clusters_held(ffn_hidden_pair_kernel<GRAD>, 2, kThreads, kSmem); });
  return held[dev & 63];
}

int matrix_map(CUtensorMap* m, const void* ptr, long long rows, long long cols, uint32_t box_rows, uint32_t box_cols) {
  const uint64_t dims[4] = {(uint64_t)cols, (uint64_t)rows, 1, 1};
  const uint64_t str[3] = {(uint64_t)cols * 2, (uint64_t)cols * 2 * rows, (uint64_t)cols * 2 * rows};
  const uint32_t box[4] = {box_cols, box_rows, 1, 1};
  return make_tmap(m, ptr, 2, 4, dims, str, box, static_cast<int>(box_cols) * 2);
}

}  // namespace

bool ffn_hidden_ok(int c, int hidden) {
  return c % 64 == 0 && hidden % 64 == 0 && pairs_held<true>() > 0 && pairs_held<false>() > 0;
}

int launch_ffn_hidden(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, void* h, void* dab, int rows, int c,
                      int hidden) {
  const bool grad = dy != nullptr;
  CUtensorMap tx, td, t1, to;
  KFB_TRY(matrix_map(&tx, x, rows, c, kRows, 64));
  KFB_TRY(matrix_map(&td, grad ? dy : x, rows, c, kRows, 64));
  KFB_TRY(matrix_map(&t1, w_in, 2ll * hidden, c, kChunk, 64));
  if (grad) {
    KFB_TRY(matrix_map(&to, w_out, c, hidden, 64, 32));
  } else {
    to = t1;
  }
  const int held = grad ? pairs_held<true>() : pairs_held<false>();
  KFB_CHECK_ARG(held > 0, "feed_forward: the device holds no pair of this kernel");
  HiddenParams p = {};
  p.rows = rows;
  p.k_blocks = c / 64;
  p.chunks = hidden / kChunk;
  p.hidden = hidden;
  p.resident = p.k_blocks <= kRowSlots;
  p.h = static_cast<__nv_bfloat16*>(h);
  p.dab = static_cast<__nv_bfloat16*>(dab);
  const int blocks = cdiv(rows, 2 * kRows);
  // few row blocks: their chunks over several pairs
  p.groups = blocks >= held ? 1 : held / blocks < p.chunks ? held / blocks : p.chunks;
  p.per_group = cdiv(p.chunks, p.groups);
  p.groups = cdiv(p.chunks, p.per_group);
  p.units = blocks * p.groups;
  LaunchScope scope(stream, grad ? "feed_forward_hidden_grad" : "feed_forward_hidden");
  return launch_kernel_clustered(stream, grad ? ffn_hidden_pair_kernel<true> : ffn_hidden_pair_kernel<false>, 2, 2 * (p.units < held ? p.units : held),
                                 kThreads, kSmem, tx, td, t1, to, p);
}

}  // namespace kfb
