// The gradient of the gated feed-forward with respect to its rows, in one kernel:
//   a, b = x Wa^T, x Wb^T,  dh = dy Wo,  da = dh b silu'(a),  db = dh silu(a),  dx = da Wa + db Wb
// for 128 or 256 channels, bf16; h, da and db are stored only where the weights' gradients want them (SPILL).
//
// What bounds it.  Five products of rows x channels x hidden channels; as separate launches da and db alone are 4 bytes per row and hidden channel
// written and read, and the memory takes writes at 4 TB/s only (measured, where a copy moves 6.5).  Here they go from one product to the next through
// tensor memory.
//
// Split.  A CTA pair takes 256 rows, 128 in each CTA, and walks the hidden channels in chunks of 64:
//   S  = [x [Wa; Wb]^T | dy Wo]   192 columns                              (CTA 0 loads the chunk's rows of Wa, CTA 1 those of Wb, each half of Wo's)
//   P  = da, db as bf16           64 columns of tensor memory, 16 hidden channels of da and db in turn
//   dX += P [Wa; Wb]              C columns, Wa and Wb read across k       (each CTA loads its half of the channels)
// S and dX have a thread each that issues them, in the order S(i + 1), dX(i): dX runs while sixteen warps bring S into registers, so that one S buffer is
// enough; with P and dX it fills the tensor memory at 256 channels.  x and dy stay in shared memory for a tile; the next tile's come into L2 meanwhile, and
// into the buffers as its slots fall free.
//
// Measured, 147 456 rows: 128 channels, 512 hidden, 84 us (59 at the measured burst rate of the products); a chunk takes 1 750 cycles, of which S is 800 and
// dX 500, the rest the way from S into registers and back to the thread that issues the next (polling there changes nothing), and a tile's end 2 200.  256 channels, 1 024 hidden, kept: 345 us, 905 MB written (3.3 TB/s with
// what is read, where writes alone reach 4; 294 without them, products 236).
#include <mutex>

#include "feed_forward_hidden.cuh"
#include "gemm.cuh"   // tanh_fast, pack_bf16x2
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int kRows = 128, kChunk = 64;
constexpr int kBox = kRows * 128;                    // [128 rows][64 bf16], 128-byte swizzle
constexpr int kRowSlot = 2 * kBox, kRowSlots = 4;    // a 64-wide block of x and of dy
constexpr int kW1 = 64 * 128, kWo = 64 * 64;         // a CTA's [64 hidden][64 k] of Wa or Wb, and [64 k][32 hidden] of Wo (64-byte swizzle)
constexpr int kWBlock = kW1 + kWo;
constexpr int kOut = 32 * 128;                       // [32 rows][64 channels] bf16 on its way out, 128-byte swizzle
constexpr int kEpiWarp = 4, kEpiWarps = 16;          // four warps for each 32 rows, 16 hidden channels each
constexpr int kThreads = 32 * (kEpiWarp + kEpiWarps);
template <int C>
struct Cfg {
  // (every wait and every commit costs the thread that issues the products some 100 cycles: few and large slots)
  static constexpr int kWSlot = 2 * kWBlock, kWSlots = 2;        // 128 k of a chunk's S
  static constexpr int kVSlot = 2 * 64 * (C / 2) * 2, kVSlots = C == 128 ? 2 : 1;   // the [2 x 64 hidden][C / 2] that dX takes of Wa and Wb
  // 128 channels: a tile's x and dy are brought into tensor memory too (128 columns).  A product whose left operand comes from shared memory takes some 40
  // cycles longer: 93 for 128 columns where it is 63 from tensor memory, 67 for 64 where it is 37 (pairs, 256 rows x 16).
  static constexpr bool kTmemRows = C == 128;
  static constexpr int kSmem = kRowSlots * kRowSlot + kWSlots * kWSlot + kVSlots * kVSlot + 4 * kOut + 512 + 1024;
  static_assert(kSmem <= 232448, "shared memory");
};

struct RowsParams {
  int rows, chunks, hidden, tiles;
};

__device__ __forceinline__ uint64_t wo_desc(uint32_t addr) {   // [k][32 hidden] rows of 64 bytes, eight of them (a swizzle atom) 512 bytes apart
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (1ull << 16) | (static_cast<uint64_t>(512 >> 4) << 32) | (1ull << 46) | (4ull << 61);
}
__device__ __forceinline__ uint64_t v_desc(uint32_t addr) {    // [64 k][64 channels] boxes of 128-byte rows, the next 64 channels a box further
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(8192 >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// The four warps that share 32 rows.
__device__ __forceinline__ void quad_sync(int quad) { asm volatile("bar.sync %0, 128;" ::"r"(quad + 1) : "memory"); }

template <int C, bool SPILL>
__global__ void __launch_bounds__(kThreads, 1)
ffn_rows_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_dy, const __grid_constant__ CUtensorMap tm_w1,
                     const __grid_constant__ CUtensorMap tm_wo, const __grid_constant__ CUtensorMap tm_dx, const __grid_constant__ CUtensorMap tm_h,
                     const __grid_constant__ CUtensorMap tm_dab, const RowsParams p) {
  constexpr int kK = C / 64, kWSlot = Cfg<C>::kWSlot, kWSlots = Cfg<C>::kWSlots, kVSlot = Cfg<C>::kVSlot, kVSlots = Cfg<C>::kVSlots;
  constexpr bool kTmemRows = Cfg<C>::kTmemRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* s_rows = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_w = s_rows + kRowSlots * kRowSlot;
  uint8_t* s_v = s_w + kWSlots * kWSlot;
  uint8_t* s_out = s_v + kVSlots * kVSlot;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_out + 4 * kOut);
  uint64_t* w_full = bars;                        // in the leader: both CTAs' copies
  uint64_t* w_free = w_full + kWSlots;
  uint64_t* v_full = w_free + kWSlots;            // in the leader
  uint64_t* v_free = v_full + kVSlots;
  uint64_t* r_full = v_free + kVSlots;            // in the leader (kTmemRows: of this CTA's rows)
  uint64_t* r_free = r_full + kRowSlots;
  uint64_t* s_full = r_free + kRowSlots;
  uint64_t* s_free = s_full + 1;                  // in the leader: the element-wise warps of both CTAs
  uint64_t* s_issued = s_free + 1;                // [2] in the leader: dX of the chunk before may follow (S may be two chunks ahead of it)
  uint64_t* p_full = s_issued + 2;                // in the leader: the element-wise warps of both CTAs
  uint64_t* p_free = p_full + 1;
  uint64_t* o_full = p_free + 1;
  uint64_t* o_free = o_full + 1;                  // in the leader, likewise
  uint64_t* xy_full = o_free + 1;                 // in the leader: x and dy of both CTAs' rows are in tensor memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(xy_full + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int tile0 = blockIdx.x >> 1, tile_step = gridDim.x >> 1;
  const int my_tiles = (p.tiles - tile0 + tile_step - 1) / tile_step;      // (the grid has no pair without a tile)
  const int total = my_tiles * p.chunks;
  auto row0_of = [&](int it) { return (2 * (tile0 + it * tile_step) + rank) * kRows; };

  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tm_x);
    ptx::prefetch_tmap(&tm_w1);
    for (int i = 0; i < kWSlots; ++i) {
      ptx::mbar_init(&w_full[i], 1);
      ptx::mbar_init(&w_free[i], 1);
    }
    for (int i = 0; i < kVSlots; ++i) {
      ptx::mbar_init(&v_full[i], 1);
      ptx::mbar_init(&v_free[i], 1);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      ptx::mbar_init(&r_full[i], 1);
      ptx::mbar_init(&r_free[i], kTmemRows ? kEpiWarps / 2 : 1);
    }
    ptx::mbar_init(xy_full, 2 * kEpiWarps);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(s_free, 2 * kEpiWarps);
    ptx::mbar_init(&s_issued[0], 1);
    ptx::mbar_init(&s_issued[1], 1);
    ptx::mbar_init(p_full, 2 * kEpiWarps);
    ptx::mbar_init(p_free, 1);
    ptx::mbar_init(o_full, 1);
    ptx::mbar_init(o_free, 2 * kEpiWarps);
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
  const uint32_t tmem = *tmem_slot, tmem_s = tmem + C, tmem_p = tmem_s + 192, tmem_xy = tmem_p + 64;      // dX first
  grid_dependency_enter();

  if (warp == 0) {
    // ---------------------------------------------------------------- weights, in the order of the products
    if (ptx::elect_one()) {
      int st = 0, v = 0;
      uint32_t ph = 0, v_ph = 0;
      bool ok = true;
      int c1 = 0, c2 = 0;
      for (int i = 0; ok && i <= total; ++i) {
        if (i < total) {
          for (int kb = 0; kb < kK; kb += 2) {
            ok = ptx::mbar_wait(&w_free[st], ph ^ 1, 541);
            if (!ok) break;
            if (rank == 0) ptx::mbar_expect_tx(&w_full[st], 2 * kWSlot);
            const uint32_t bar = ptx::leader_addr(&w_full[st]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint8_t* d = s_w + st * kWSlot + q * kWBlock;
              ptx::tma_load_4d_pair(d, &tm_w1, bar, (kb + q) * 64, rank * p.hidden + c1 * kChunk, 0, 0);
              ptx::tma_load_4d_pair(d + kW1, &tm_wo, bar, c1 * kChunk + rank * 32, (kb + q) * 64, 0, 0);
            }
            if (++st == kWSlots) { st = 0; ph ^= 1u; }
          }
          if (++c1 == p.chunks) c1 = 0;
        }
        if (i > 0) {
          ok = ok && ptx::mbar_wait(&v_free[v], v_ph ^ 1, 542);
          if (!ok) break;
          if (rank == 0) ptx::mbar_expect_tx(&v_full[v], 2 * kVSlot);
          const uint32_t bar = ptx::leader_addr(&v_full[v]);
#pragma unroll
          for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int q = 0; q < C / 128; ++q)
              ptx::tma_load_4d_pair(s_v + v * kVSlot + which * (kVSlot / 2) + q * 8192, &tm_w1, bar, rank * (C / 2) + q * 64,
                                    which * p.hidden + c2 * kChunk, 0, 0);
          if (++v == kVSlots) { v = 0; v_ph ^= 1u; }
          if (++c2 == p.chunks) c2 = 0;
        }
      }
      // the last products' arrivals at this CTA's barriers, before it may exit
      for (int i = 0; ok && i < kWSlots; ++i) {
        ok = ptx::mbar_wait(&w_free[st], ph ^ 1, 543);
        if (++st == kWSlots) { st = 0; ph ^= 1u; }
      }
      for (int i = 0; ok && i < kVSlots; ++i) {
        ok = ptx::mbar_wait(&v_free[v], v_ph ^ 1, 544);
        if (++v == kVSlots) { v = 0; v_ph ^= 1u; }
      }
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- rows
    if (ptx::elect_one()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int it = 0; ok && it < my_tiles; ++it) {
        for (int kb = 0; kb < kK; ++kb) {
          ok = ptx::mbar_wait(&r_free[st], ph ^ 1, 545);
          if (!ok) break;
          if constexpr (kTmemRows) {
            ptx::mbar_expect_tx(&r_full[st], kRowSlot);
            ptx::tma_load_4d(s_rows + st * kRowSlot, &tm_x, &r_full[st], kb * 64, row0_of(it), 0, 0);
            ptx::tma_load_4d(s_rows + st * kRowSlot + kBox, &tm_dy, &r_full[st], kb * 64, row0_of(it), 0, 0);
          } else {
            if (rank == 0) ptx::mbar_expect_tx(&r_full[st], 2 * kRowSlot);
            const uint32_t bar = ptx::leader_addr(&r_full[st]);
            ptx::tma_load_4d_pair(s_rows + st * kRowSlot, &tm_x, bar, kb * 64, row0_of(it), 0, 0);
            ptx::tma_load_4d_pair(s_rows + st * kRowSlot + kBox, &tm_dy, bar, kb * 64, row0_of(it), 0, 0);
          }
          if (++st == kRowSlots) { st = 0; ph ^= 1u; }
        }
        if (it + 1 < my_tiles)
          for (int kb = 0; kb < kK; ++kb) {
            ptx::tma_prefetch_4d(&tm_x, kb * 64, row0_of(it + 1), 0, 0);
            ptx::tma_prefetch_4d(&tm_dy, kb * 64, row0_of(it + 1), 0, 0);
          }
      }
      for (int i = 0; ok && i < kRowSlots; ++i) {
        ok = ptx::mbar_wait(&r_free[st], ph ^ 1, 546);
        if (++st == kRowSlots) { st = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- S
    if (rank == 0 && ptx::elect_one()) {
      constexpr uint32_t idesc_s = ptx::make_idesc(2 * kRows, 2 * kChunk, 1), idesc_g = ptx::make_idesc(2 * kRows, kChunk, 1) | (1u << 16);
      const uint64_t row_desc = ptx::make_kmajor_desc<128>(ptx::smem_u32(s_rows));
      const uint64_t w1_desc = ptx::make_kmajor_desc<128>(ptx::smem_u32(s_w)), g_desc = wo_desc(ptx::smem_u32(s_w) + kW1);
      int st = 0, rs0 = 0, c = 0, it = 0;
      uint32_t ph = 0, r_ph = 0;
      bool ok = true;
      for (int i = 0; ok && i < total; ++i) {
        ok = ptx::mbar_wait(s_free, (i & 1) ^ 1, 547, ptx::kPolls);
        if (kTmemRows && c == 0) ok = ok && ptx::mbar_wait(xy_full, it & 1, 557, ptx::kPolls);
        if (!ok) break;
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int kb = 0; kb < kK; ++kb) {
          const int rs = rs0 + kb;                  // (kRowSlots is a multiple of kK)
          if (!kTmemRows && c == 0) ok = ptx::mbar_wait(&r_full[rs], r_ph, 548, ptx::kPolls);
          if ((kb & 1) == 0) ok = ok && ptx::mbar_wait(&w_full[st], ph, 549, ptx::kPolls);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const uint32_t w_at = st * (kWSlot >> 4) + (kb & 1) * (kWBlock >> 4);
          const uint64_t xd = row_desc + rs * (kRowSlot >> 4), wd = w1_desc + w_at, gd = g_desc + w_at;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (kTmemRows) ptx::mma_f16_ts_pair(tmem_s, tmem_xy + kb * 32 + k * 8, wd + k * 2, idesc_s, kb > 0 || k > 0 ? 1u : 0u);
            else ptx::mma_f16_ss_pair(tmem_s, xd + k * 2, wd + k * 2, idesc_s, kb > 0 || k > 0 ? 1u : 0u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (kTmemRows)
              ptx::mma_f16_ts_pair(tmem_s + 128, tmem_xy + 64 + kb * 32 + k * 8, gd + k * (1024 >> 4), idesc_g, kb > 0 || k > 0 ? 1u : 0u);
            else ptx::mma_f16_ss_pair(tmem_s + 128, xd + (kBox >> 4) + k * 2, gd + k * (1024 >> 4), idesc_g, kb > 0 || k > 0 ? 1u : 0u);
          }
          if (!kTmemRows && c == p.chunks - 1) ptx::tc_commit_pair(&r_free[rs]);
          if (kb & 1) {
            ptx::tc_commit_pair(&w_free[st]);
            if (++st == kWSlots) { st = 0; ph ^= 1u; }
          }
        }
        if (!ok) break;
        ptx::tc_commit_pair(s_full);
        ptx::mbar_arrive(&s_issued[i & 1]);
        if (++c == p.chunks) {
          c = 0;
          ++it;
          rs0 += kK;
          if (rs0 == kRowSlots) { rs0 = 0; r_ph ^= 1u; }
        }
      }
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- dX
    if (rank == 0 && ptx::elect_one()) {
      constexpr uint32_t idesc = ptx::make_idesc(2 * kRows, C, 1) | (1u << 16);
      const uint64_t vd0 = v_desc(ptx::smem_u32(s_v));
      int v = 0, c = 0, it = 0;
      uint32_t v_ph = 0;
      bool ok = true;
      for (int i = 0; ok && i < total; ++i) {
        if (c == 0) ok = ptx::mbar_wait(o_free, (it & 1) ^ 1, 550, ptx::kPolls);
        // (behind the next chunk's S, not before or within it: the tensor core then has dX to do while that S is read)
        if (i + 1 < total) ok = ok && ptx::mbar_wait(&s_issued[(i + 1) & 1], ((i + 1) >> 1) & 1, 556, ptx::kPolls);
        ok = ok && ptx::mbar_wait(p_full, i & 1, 551, ptx::kPolls);
        ok = ok && ptx::mbar_wait(&v_full[v], v_ph, 552, ptx::kPolls);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint64_t vd = vd0 + v * (kVSlot >> 4);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          ptx::mma_f16_ts_pair(tmem, tmem_p + (k >> 2) * 8 + (k & 3) * 16, vd + (k >> 2) * (kVSlot >> 5) + (k & 3) * (2048 >> 4), idesc,
                               c > 0 || k > 0 ? 1u : 0u);
        ptx::tc_commit_pair(&v_free[v]);
        if (++v == kVSlots) { v = 0; v_ph ^= 1u; }
        ptx::tc_commit_pair(p_free);
        if (++c == p.chunks) {
          ptx::tc_commit_pair(o_full);
          c = 0;
          ++it;
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- da, db (and h); dx
    const int part = (warp - kEpiWarp) >> 2, quad = warp & 3;
    const uint32_t t_quad = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem_s + t_quad + part * 16, t_p = tmem_p + t_quad + part * 16, t_o = tmem + t_quad;
    bool ok = true;
    // 16 channels of a row from each of the four warps, as one box by the copy engine: stores from registers are 32-byte sectors of 32 lines each, which left
    // an SM at 10 bytes a cycle and held the warps up.  (Where a wait gave up the warps keep meeting here, and leave memory alone.)
    uint8_t* box = s_out + quad * kOut;
    // 16-byte cells of a row's 128 bytes, swizzled: cell j of row r lies at j ^ (r % 8)
    uint4 *cell0 = reinterpret_cast<uint4*>(box + lane * 128 + (((2 * part) ^ (lane & 7)) << 4));
    uint4 *cell1 = reinterpret_cast<uint4*>(box + lane * 128 + (((2 * part + 1) ^ (lane & 7)) << 4));
    const bool sender = part == 0 && lane == 0;
    auto send = [&](const CUtensorMap* map, const uint32_t (&w)[8], int col, int row) {
      if (sender) ptx::tma_store_wait_read();      // the box that left last
      quad_sync(quad);
      *cell0 = make_uint4(w[0], w[1], w[2], w[3]);
      *cell1 = make_uint4(w[4], w[5], w[6], w[7]);
      ptx::fence_proxy_async_smem();
      quad_sync(quad);
      if (sender && ok && row < p.rows) {
        ptx::tma_store_4d(map, box, col, row, 0, 0);
        ptx::tma_store_commit();
      }
    };
    // the finished tile's dx
    auto finish = [&](int it) {
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(o_full, it & 1, 553)) != 0;
      ptx::tc_fence_after_sync();
      uint32_t w[C / 64][8];
#pragma unroll
      for (int q = 0; q < C / 64; ++q) {
        uint32_t o[16];
        ptx::tmem_ld_32x32b_x16(t_o + q * 64 + part * 16, o);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j) w[q][j] = pack_bf16x2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]));
      }
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::leader_addr(o_free));
#pragma unroll
      for (int q = 0; q < C / 64; ++q) send(&tm_dx, w[q], q * 64, row0_of(it) + quad * 32);
    };
    // da (at = 0) or db (8) of the last chunk, which P still holds
    auto keep = [&](int at, int col, int row) {
      uint32_t w[8];
      ptx::tmem_ld_32x32b_x8(t_p + at, w);
      ptx::tmem_ld_wait();
      send(&tm_dab, w, col, row);
    };
    // a tile's x and dy into tensor memory: a block of 64 channels of one of them a warp
    auto take = [&](int it) {
      const int slot = (2 * it + (part & 1)) & 3;
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(&r_full[slot], (it >> 1) & 1, 558)) != 0;
      const int r = quad * 32 + lane;
      const uint8_t* src = s_rows + slot * kRowSlot + (part >> 1) * kBox + r * 128;
      uint32_t w[2][16];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint4 v = *reinterpret_cast<const uint4*>(src + ((j ^ (r & 7)) << 4));
        w[j >> 2][4 * (j & 3)] = v.x;
        w[j >> 2][4 * (j & 3) + 1] = v.y;
        w[j >> 2][4 * (j & 3) + 2] = v.z;
        w[j >> 2][4 * (j & 3) + 3] = v.w;
      }
      ptx::tmem_st_32x32b_x16(tmem_xy + t_quad + (part >> 1) * 64 + (part & 1) * 32, w[0]);
      ptx::tmem_st_32x32b_x16(tmem_xy + t_quad + (part >> 1) * 64 + (part & 1) * 32 + 16, w[1]);
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(&r_free[slot]);
        ptx::mbar_arrive_cluster(ptx::leader_addr(xy_full));
      }
    };
    if constexpr (kTmemRows) take(0);
    int c = 0, it = 0, last_col = 0, last_row = 0;
    for (int i = 0; i < total; ++i) {
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(s_full, i & 1, 554)) != 0;
      ptx::tc_fence_after_sync();
      uint32_t a[16], b[16], g[16];
      ptx::tmem_ld_32x32b_x16(t_s, a);
      ptx::tmem_ld_32x32b_x16(t_s + 64, b);
      ptx::tmem_ld_32x32b_x16(t_s + 128, g);
      ptx::tmem_ld_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::leader_addr(s_free));
      // (the tile's last S is complete: the next tile's rows may take its operands' place)
      if (kTmemRows && c == p.chunks - 1 && it + 1 < my_tiles) take(it + 1);
      uint32_t hw[8], aw[8], bw[8];
      auto pairs = [&](int j0) {
#pragma unroll
        for (int j = j0; j < j0 + 8; j += 2) {
          // s = tanh(a / 2) / 2 + 1 / 2, silu = a s, silu' = s + silu (1 - s)
          const uint64_t half2 = ptx::pack2(0.5f, 0.5f), one2 = ptx::pack2(1.0f, 1.0f), minus2 = ptx::pack2(-1.0f, -1.0f);
          const uint64_t av = ptx::pack2(a[j], a[j + 1]), bv = ptx::pack2(b[j], b[j + 1]), gv = ptx::pack2(g[j], g[j + 1]);
          const float2 ah = ptx::unpack2(ptx::mul2(av, half2));
          const uint64_t sv = ptx::fma2(ptx::pack2(tanh_fast(ah.x), tanh_fast(ah.y)), half2, half2);
          const uint64_t silu = ptx::mul2(av, sv);
          const uint64_t slope = ptx::fma2(silu, ptx::fma2(sv, minus2, one2), sv);
          aw[j >> 1] = pack_bf16x2(ptx::mul2(ptx::mul2(gv, bv), slope));
          bw[j >> 1] = pack_bf16x2(ptx::mul2(gv, silu));
          if (SPILL) hw[j >> 1] = pack_bf16x2(ptx::mul2(silu, bv));
        }
      };
      // (the last chunk's da and db leave between the halves of this one's arithmetic: a box takes some 500 cycles to go)
      if (SPILL && i > 0) keep(0, last_col, last_row);
      pairs(0);
      if (SPILL && i > 0) keep(8, p.hidden + last_col, last_row);
      pairs(8);
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(p_free, (i & 1) ^ 1, 555)) != 0;
      ptx::tc_fence_after_sync();
      ptx::tmem_st_32x32b_x8(t_p, aw);
      ptx::tmem_st_32x32b_x8(t_p + 8, bw);
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::leader_addr(p_full));
      if (SPILL) {
        last_col = c * kChunk;
        last_row = row0_of(it) + quad * 32;
        send(&tm_h, hw, last_col, last_row);
      }
      // (behind the next tile's first chunk: its S then runs under dX of the last)
      if (c == 0 && it > 0) finish(it - 1);
      if (++c == p.chunks) {
        c = 0;
        ++it;
      }
    }
    if (SPILL) {
      keep(0, last_col, last_row);
      keep(8, p.hidden + last_col, last_row);
    }
    finish(my_tiles - 1);
    if (sender) ptx::tma_store_wait_all();
  }

  ptx::tc_fence_before_sync();
  __syncwarp();
  ptx::cluster_sync();      // neither CTA leaves while the other may still read its operands or reach its barriers
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc_pair(tmem, 512);
  }
}

template <int C, bool SPILL>
int pairs_held() {
  static std::once_flag once[64];
  static int held[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  std::call_once(once[dev & 63], [&] { held[dev & 63] = clusters_held(ffn_rows_pair_kernel<C, SPILL>, 2, kThreads, Cfg<C>::kSmem); });
  return held[dev & 63];
}

int matrix_map(CUtensorMap* m, const void* ptr, long long rows, long long cols, uint32_t box_rows, uint32_t box_cols) {
  const uint64_t dims[4] = {(uint64_t)cols, (uint64_t)rows, 1, 1};
  const uint64_t str[3] = {(uint64_t)cols * 2, (uint64_t)cols * 2 * rows, (uint64_t)cols * 2 * rows};
  const uint32_t box[4] = {box_cols, box_rows, 1, 1};
  return make_tmap(m, ptr, 2, 4, dims, str, box, static_cast<int>(box_cols) * 2);
}

template <int C, bool SPILL>
int launch(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, void* dx, void* h, void* dab, int rows,
           int hidden) {
  CUtensorMap tx, td, t1, to, tdx, th, tg;
  KFB_TRY(matrix_map(&tx, x, rows, C, kRows, 64));
  KFB_TRY(matrix_map(&td, dy, rows, C, kRows, 64));
  KFB_TRY(matrix_map(&t1, w_in, 2ll * hidden, C, kChunk, 64));
  KFB_TRY(matrix_map(&to, w_out, C, hidden, 64, 32));
  KFB_TRY(matrix_map(&tdx, dx, rows, C, 32, 64));
  th = tg = tdx;
  if (SPILL) {
    KFB_TRY(matrix_map(&th, h, rows, hidden, 32, 64));
    KFB_TRY(matrix_map(&tg, dab, rows, 2ll * hidden, 32, 64));
  }
  const int held = pairs_held<C, SPILL>();
  KFB_CHECK_ARG(held > 0, "feed_forward: the device holds no pair of this kernel");
  RowsParams p = {};
  p.rows = rows;
  p.chunks = hidden / kChunk;
  p.hidden = hidden;
  p.tiles = cdiv(rows, 2 * kRows);
  LaunchScope scope(stream, SPILL ? "feed_forward_rows_grad_kept" : "feed_forward_rows_grad");
  return launch_kernel_clustered(stream, ffn_rows_pair_kernel<C, SPILL>, 2, 2 * (p.tiles < held ? p.tiles : held), kThreads, Cfg<C>::kSmem, tx, td, t1,
                                 to, tdx, th, tg, p);
}

}  // namespace

bool ffn_rows_ok(int c, int hidden) {
  if (hidden % kChunk != 0) return false;
  return c == 128 ? pairs_held<128, false>() > 0 : c == 256 && pairs_held<256, false>() > 0 && pairs_held<256, true>() > 0;
}

int launch_ffn_rows(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, void* dx, void* h, void* dab, int rows,
                    int c, int hidden) {
  if (c == 128) {
    KFB_CHECK_ARG(h == nullptr, "feed_forward: 128 channels keep nothing");
    return launch<128, false>(stream, x, dy, w_in, w_out, dx, h, dab, rows, hidden);
  }
  return h != nullptr ? launch<256, true>(stream, x, dy, w_in, w_out, dx, h, dab, rows, hidden)
                      : launch<256, false>(stream, x, dy, w_in, w_out, dx, h, dab, rows, hidden);
}

}  // namespace kfb
