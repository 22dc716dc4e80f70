// D[m][n] = sum_k A(m, k) B(n, k) for operands stored along k or across it (see matmul.cuh).
//
// A CTA computes one 128 x 128 tile of one piece of k of one of up to three products: a thread fetches 64-wide blocks of both operands with TMA into a ring, a thread issues
// the products, four warps bring the accumulator from tensor memory to global memory.  Two CTAs share an SM, so that one's start and end lie
// under the other's products.  An operand stored across k ([k][i]) is fetched as two boxes of 64 k by 64 i and read MN-major as it lies: the
// gradients of weights contract over rows, and nothing is transposed for them.
// What bounds it: reading the left operand from shared memory costs a product 40 cycles where its multiplications take 64, and short contractions their
// start and end (some 3 us).  331 rows of 384 channels, 1 536 hidden ones: dx and the weights' gradients, 2.3 GFLOP, in one launch of 9 us.  Many rows of
// the usual widths have kernels of their own.
// fp32-accurate mode: three parts an operand, six products, x0 w0 in an accumulator of its own (the tensor core cuts off relative to the
// accumulator at every step: the five small ones keep their small error apart).  That cut goes with the length of the contraction, 1e-6 of the result after 1 024: `turns`
// accumulators that take the blocks of k in turn are smaller and are cut a third as often each (3e-7; float32 sums one after the other 6e-7).  A CTA has an SM, and its tensor memory, to itself.
#include "matmul.cuh"

#include "gemm.cuh"   // split3, epi_store_chunk
#include "linear_tail.cuh"
#include "ops_common.cuh"
#include "ptx.cuh"

namespace kfb {
namespace {

constexpr int kTile = 128, kK = 64;
constexpr int kOperand = kTile * kK * 2;           // bytes of a block of one operand
constexpr int kStage = 2 * kOperand;
constexpr int kThreads = 192;                      // TMA, products, four warps of rows

struct MmParams {
  int m, n, m_tiles, n_tiles, splits;
  int blocks, per_split;                           // of 64 along k: all, of a piece
  int a_by_k, b_by_k;
  EpiSeg out;
  long long plane_d;
  int accumulate;
};
struct MmBatch {
  CUtensorMap a[kMostMatmuls], b[kMostMatmuls];
  MmParams p[kMostMatmuls];
  MatmulTail tail;                                 // of a launch of one product
  int turns;                                       // PARTS = 3
  int end[kMostMatmuls];                           // blocks of the grid up to and with each product
};

template <int PARTS>
constexpr int stages() { return PARTS == 3 ? 6 : 3; }
template <int PARTS>
constexpr int smem_bytes() { return stages<PARTS>() * kStage + 1024 + 256; }

__device__ __forceinline__ uint64_t by_k_desc(uint32_t addr) {
  // 128-byte swizzled rows of 64 i, one per k: eight of them (a swizzle atom) 1024 bytes apart, the next 64 i half an operand further
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>((kOperand / 2) >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// The launches with a tail have tiles of 64 columns and twice the warps for them: few rows make few tiles, and a tile's tail is the longer part.
template <bool TAIL>
constexpr int tile_columns() { return TAIL ? 64 : kTile; }
template <bool TAIL>
constexpr int threads() { return TAIL ? kThreads + 128 : kThreads; }

// A tail's tensor at eight neighbouring columns, as pairs of float32.
__device__ __forceinline__ void tail_load(const void* p, long long o, int fp32, uint64_t (&v)[4]) {
  if (fp32) {
    const ulonglong2* q = reinterpret_cast<const ulonglong2*>(static_cast<const float*>(p) + o);
    const ulonglong2 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + o);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ptx::pack2(w[i] << 16, w[i] & 0xffff0000u);
  }
}

// 32 columns of a row through the tail.  x: aux there, zeros where there is none.  (Columns end at a multiple of 8, the tensors' rows start on 16-byte boundaries.)
__device__ __forceinline__ void tail_chunk(const MatmulTail& t, const EpiSeg& out, long long plane, long long row_off, int row_group, int col, int n, const float (&v)[32],
                                           const uint64_t (&x)[4][4], bool there, int lane) {
  with_activation(t.act, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int at = col + 8 * c;
      if (at >= n) break;
      uint64_t z[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = ptx::pack2(v[8 * c + 2 * i], v[8 * c + 2 * i + 1]);
      if (t.bias != nullptr) {
        tail_load(t.bias, at, 1, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = ptx::add2(z[i], b[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = t.backward ? ptx::mul2(x[c][i], slope<ACT>(z[i])) : ptx::add2(activation<ACT>(z[i]), x[c][i]);
      if (t.partial != nullptr) {
        const float s = sum_rows8(z, lane);
        if ((lane & 3) == 0) t.partial[static_cast<long long>(row_group) * n + at + 4 * (lane >> 4 & 1) + 2 * (lane >> 3 & 1) + (lane >> 2 & 1)] = s;
      }
      if (!there) continue;
      if (t.parts == 3) {
        __nv_bfloat16 q[3][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = ptx::unpack2(z[i]);
          split3(f.x, q[0][2 * i], q[1][2 * i], q[2][2 * i]);
          split3(f.y, q[0][2 * i + 1], q[1][2 * i + 1], q[2][2 * i + 1]);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out.dst) + k * plane + row_off + at) = *reinterpret_cast<const uint4*>(q[k]);
      } else if (out.out_fp32) {
        ulonglong2* d = reinterpret_cast<ulonglong2*>(static_cast<float*>(out.dst) + row_off + at);
        d[0] = make_ulonglong2(z[0], z[1]);
        d[1] = make_ulonglong2(z[2], z[3]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out.dst) + row_off + at) = make_uint4(pack_bf16x2(z[0]), pack_bf16x2(z[1]), pack_bf16x2(z[2]), pack_bf16x2(z[3]));
      }
    }
  });
}

template <int PARTS, bool TAIL>
__global__ void __launch_bounds__(threads<TAIL>(), PARTS == 3 ? 1 : 2) matmul_kernel(const __grid_constant__ MmBatch batch) {
  constexpr int kStages = stages<PARTS>(), kTileN = tile_columns<TAIL>(), kBytes = kOperand + kTileN * kK * 2;
  // columns of the large products' accumulators, and behind the first of the small ones'
  constexpr uint32_t kCols = PARTS == 3 ? 512 : 128;
  auto large = [](int turn) { return static_cast<uint32_t>(turn == 0 ? 0 : 128 + 128 * turn); };
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * kStage);
  uint64_t* empty = full + kStages;
  uint64_t* done = empty + kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int which = 0, block = blockIdx.x;
#pragma unroll
  for (int i = 0; i + 1 < kMostMatmuls; ++i)
    if (static_cast<int>(blockIdx.x) >= batch.end[i]) {
      which = i + 1;
      block = blockIdx.x - batch.end[i];
    }
  const MmParams& p = batch.p[which];
  const CUtensorMap &tm_a = batch.a[which], &tm_b = batch.b[which];
  const int m_tile = block % p.m_tiles, n_tile = block / p.m_tiles % p.n_tiles, split = block / (p.m_tiles * p.n_tiles);
  const int first = split * p.per_split, last = min(first + p.per_split, p.blocks);
  if (threadIdx.x == 0) {
    ptx::prefetch_tmap(&tm_a);
    ptx::prefetch_tmap(&tm_b);
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], 1);
    }
    ptx::mbar_init(done, 1);
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, kCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_enter();

  if (warp == 0) {
    if (ptx::elect_one()) {
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = first; ok && kb < last; ++kb)
        for (int part = 0; part < PARTS; ++part) {
          ok = ptx::mbar_wait(&empty[st], ph ^ 1, 501);
          if (!ok) break;
          ptx::mbar_expect_tx(&full[st], kBytes);
          uint8_t *a = ring + st * kStage, *b = a + kOperand;
          if (p.a_by_k) {
            ptx::tma_load_3d(a, &tm_a, &full[st], m_tile * kTile, kb * kK, part);
            ptx::tma_load_3d(a + kOperand / 2, &tm_a, &full[st], m_tile * kTile + 64, kb * kK, part);
          } else {
            ptx::tma_load_3d(a, &tm_a, &full[st], kb * kK, m_tile * kTile, part);
          }
          if (p.b_by_k) {                            // (never with a tail)
            ptx::tma_load_3d(b, &tm_b, &full[st], n_tile * kTileN, kb * kK, part);
            ptx::tma_load_3d(b + kOperand / 2, &tm_b, &full[st], n_tile * kTileN + 64, kb * kK, part);
          } else {
            ptx::tma_load_3d(b, &tm_b, &full[st], kb * kK, n_tile * kTileN, part);
          }
          if (++st == kStages) { st = 0; ph ^= 1u; }
        }
    }
  } else if (warp == 1) {
    if (ptx::elect_one()) {
      const uint32_t idesc = ptx::make_idesc(kTile, kTileN, 1) | (p.a_by_k ? 1u << 15 : 0u) | (p.b_by_k ? 1u << 16 : 0u);
      const uint32_t a_step = p.a_by_k ? 2048 >> 4 : 2, b_step = p.b_by_k ? 2048 >> 4 : 2;     // of 16 k
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = first; ok && kb < last; ++kb) {
        uint64_t ad[PARTS], bd[PARTS];
        int used[PARTS];
        auto product = [&](int i, int j, uint32_t d, bool fresh) {
#pragma unroll
          for (int k = 0; k < kK / 16; ++k) ptx::mma_f16_ss(d, ad[i] + k * a_step, bd[j] + k * b_step, idesc, fresh && k == 0 ? 0u : 1u);
        };
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          ok = ok && ptx::mbar_wait(&full[st], ph, 502);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const uint32_t at = ptx::smem_u32(ring + st * kStage);
          ad[i] = p.a_by_k ? by_k_desc(at) : ptx::make_kmajor_desc<128>(at);
          bd[i] = p.b_by_k ? by_k_desc(at + kOperand) : ptx::make_kmajor_desc<128>(at + kOperand);
          used[i] = st;
          if (++st == kStages) { st = 0; ph ^= 1u; }
          if (i == 0) {
            if (PARTS == 3) product(0, 0, tmem + large((kb - first) % batch.turns), kb - first < batch.turns);
            else product(0, 0, tmem, kb == first);
          } else {
            product(0, i, tmem + 128, kb == first && i == 1);
            product(i, 0, tmem + 128, false);
            if (i == 1) product(1, 1, tmem + 128, false);
          }
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) ptx::tc_commit(&empty[used[i]]);
      }
      if (ok) ptx::tc_commit(done);
    }
  } else {
    const int quad = warp & 3, row = m_tile * kTile + quad * 32 + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const long long row_off = static_cast<long long>(row) * p.out.s_n + (TAIL ? 0 : split * p.plane_d);
    // a tail's warp has 32 columns; what is added or multiplied comes while the products are made
    const int c_first = TAIL ? (warp - 2) / 4 * 32 : 0, c_end = TAIL ? c_first + 32 : kTile;
    uint64_t x[4][4];
    if constexpr (TAIL) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = n_tile * kTileN + c_first + 8 * c;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][i] = 0;
        if (batch.tail.aux != nullptr && row < p.m && at < p.n) tail_load(batch.tail.aux, row_off + at, batch.tail.aux_fp32, x[c]);
      }
    }
    const bool ok = __all_sync(0xffffffffu, ptx::mbar_wait(done, 0, 503)) != 0;
    ptx::tc_fence_after_sync();
    if (ok) {
#pragma unroll 1
      for (int c = c_first; c < c_end; c += 32) {
        const int col = n_tile * kTileN + c;
        if (col >= p.n) break;
        uint32_t raw[32];
        float v[32];
        ptx::tmem_ld_32x32b_x32(t_row + c, raw);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]);
        if (PARTS == 3) {
          for (int turn = 1; turn < batch.turns && turn < last - first; ++turn) {
            ptx::tmem_ld_32x32b_x32(t_row + large(turn) + c, raw);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(raw[i]);
          }
          ptx::tmem_ld_32x32b_x32(t_row + 128 + c, raw);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(raw[i]);
        }
        if constexpr (TAIL) {
          tail_chunk(batch.tail, p.out, p.plane_d, row_off, m_tile * 4 + quad, col, p.n, v, x, row < p.m, lane);
          continue;
        }
        if (p.accumulate && row < p.m) {
          const float* d = static_cast<const float*>(p.out.dst) + row_off + col;
          if (p.out.vec && col + 32 <= p.n) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 t = *reinterpret_cast<const float4*>(d + i);
              v[i] += t.x;
              v[i + 1] += t.y;
              v[i + 2] += t.z;
              v[i + 3] += t.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col + i < p.n) v[i] += d[i];
          }
        }
        epi_store_chunk(p.out, row_off, col, v, row < p.m);
      }
    }
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, kCols);
  }
}

int operand_map(CUtensorMap* map, const MatOperand& o, int extent, long long k, int parts, int tile) {
  const uint64_t dims[3] = {static_cast<uint64_t>(o.by_k ? extent : k), static_cast<uint64_t>(o.by_k ? k : extent), static_cast<uint64_t>(parts)};
  const uint64_t str[2] = {static_cast<uint64_t>(o.ld) * 2, static_cast<uint64_t>(parts > 1 ? o.plane : o.ld) * 2};
  const uint32_t box[3] = {64, o.by_k ? 64u : static_cast<uint32_t>(tile), 1};
  return make_tmap(map, o.ptr, 2, 3, dims, str, box, 128);
}

struct SumBatch {
  PlaneSum s[kMostMatmuls];
  unsigned end[kMostMatmuls];                      // blocks of the grid up to and with each sum
};
__global__ void __launch_bounds__(256) sum_planes_kernel(const SumBatch batch) {
  grid_dependency_enter();
  int which = 0;
  unsigned block = blockIdx.x;
#pragma unroll
  for (int i = 0; i + 1 < kMostMatmuls; ++i)
    if (blockIdx.x >= batch.end[i]) {
      which = i + 1;
      block = blockIdx.x - batch.end[i];
    }
  const PlaneSum& q = batch.s[which];
  const long long i = (static_cast<long long>(block) * 256 + threadIdx.x) * 4;
  if (i >= q.n) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < q.splits; ++k) {
    const float4 t = *reinterpret_cast<const float4*>(q.planes + k * q.plane + i);
    s.x += t.x;
    s.y += t.y;
    s.z += t.z;
    s.w += t.w;
  }
  if (q.out_fp32) *reinterpret_cast<float4*>(static_cast<float*>(q.out) + i) = s;
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(q.out) + i) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

__global__ void __launch_bounds__(256) split_planes_kernel(const float* x, __nv_bfloat16* parts, long long plane, long long n) {
  grid_dependency_enter();
  const long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const float4 v = *reinterpret_cast<const float4*>(x + i);
  const float f[4] = {v.x, v.y, v.z, v.w};
  __nv_bfloat16 q[3][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) split3(f[k], q[0][k], q[1][k], q[2][k]);
#pragma unroll
  for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(parts + k * plane + i) = *reinterpret_cast<const uint2*>(q[k]);
}

}  // namespace

int launch_matmuls(cudaStream_t stream, const MatmulArgs* list, int count, const char* tag) {
  KFB_CHECK_ARG(count >= 1 && count <= kMostMatmuls, "matmul: %d products", count);
  MmBatch batch = {};
  int blocks = 0;
  for (int i = 0; i < count; ++i) {
    const MatmulArgs& a = list[i];
    KFB_CHECK_ARG(a.m > 0 && a.n > 0 && a.k > 0 && a.k < (1ll << 31) && a.splits >= 1, "matmul: m %d n %d k %lld, %d pieces", a.m, a.n, a.k, a.splits);
    KFB_CHECK_ARG(a.out_fp32 || (a.splits == 1 && !a.accumulate), "matmul: pieces and sums need an fp32 result");
    KFB_CHECK_ARG(a.precise == list[0].precise && a.turns == list[0].turns && a.turns >= 0 && a.turns <= kMostTurns, "matmul: products of both modes in one launch, or %d turns", a.turns);
    MmParams& p = batch.p[i];
    p.m = a.m;
    p.n = a.n;
    p.m_tiles = cdiv(a.m, kTile);
    const int columns = a.tail != nullptr ? tile_columns<true>() : tile_columns<false>();
    p.n_tiles = cdiv(a.n, columns);
    p.splits = a.splits;
    p.blocks = static_cast<int>((a.k + kK - 1) / kK);
    p.per_split = cdiv(p.blocks, a.splits);
    KFB_CHECK_ARG(cdiv(p.blocks, p.per_split) == a.splits, "matmul: an empty piece of k (%d blocks in %d)", p.blocks, a.splits);
    p.a_by_k = a.a.by_k;
    p.b_by_k = a.b.by_k;
    p.out = row_major_seg(a.d, a.n, a.ld_d, 0, 0, a.out_fp32);
    if (a.splits > 1 && a.plane_d % 4 != 0) p.out.vec = 0;
    if (a.tail != nullptr) {
      KFB_CHECK_ARG(count == 1 && a.splits == 1 && !a.accumulate && !a.b.by_k && a.n % 8 == 0 && a.ld_d % 8 == 0 && a.plane_d % 8 == 0, "matmul: a tail of %d products, %d pieces, %d columns",
                    count, a.splits, a.n);
      batch.tail = *a.tail;
    }
    p.plane_d = a.plane_d;
    p.accumulate = a.accumulate;
    KFB_TRY(operand_map(&batch.a[i], a.a, a.m, a.k, a.precise ? 3 : 1, kTile));
    KFB_TRY(operand_map(&batch.b[i], a.b, a.n, a.k, a.precise ? 3 : 1, columns));
    const long long add = static_cast<long long>(p.m_tiles) * p.n_tiles * p.splits;
    KFB_CHECK_ARG(add + blocks < (1ll << 31), "matmul: %lld tiles", add);
    blocks += static_cast<int>(add);
    batch.end[i] = blocks;
  }
  for (int i = count; i < kMostMatmuls; ++i) batch.end[i] = blocks;
  batch.turns = list[0].turns > 0 ? list[0].turns : 1;
  LaunchScope scope(stream, tag);
  auto run = [&](auto kernel_of, int smem) { return launch_kernel(stream, kernel_of, blocks, list[0].tail != nullptr ? threads<true>() : threads<false>(), smem, batch); };
  if (list[0].precise) {
    if (list[0].tail != nullptr) {
      KFB_TRY((allow_smem<matmul_kernel<3, true>>(smem_bytes<3>())));
      return run(matmul_kernel<3, true>, smem_bytes<3>());
    }
    KFB_TRY((allow_smem<matmul_kernel<3, false>>(smem_bytes<3>())));
    return run(matmul_kernel<3, false>, smem_bytes<3>());
  }
  if (list[0].tail != nullptr) {
    KFB_TRY((allow_smem<matmul_kernel<1, true>>(smem_bytes<1>())));
    return run(matmul_kernel<1, true>, smem_bytes<1>());
  }
  KFB_TRY((allow_smem<matmul_kernel<1, false>>(smem_bytes<1>())));
  return run(matmul_kernel<1, false>, smem_bytes<1>());
}

int launch_sum_planes(cudaStream_t stream, const PlaneSum* list, int count) {
  KFB_CHECK_ARG(count >= 1 && count <= kMostMatmuls, "sum_planes: %d sums", count);
  SumBatch batch = {};
  unsigned blocks = 0;
  for (int i = 0; i < kMostMatmuls; ++i) {
    if (i < count) {
      KFB_CHECK_ARG(list[i].n % 4 == 0 && list[i].plane % 4 == 0, "sum_planes: %lld elements, planes %lld apart (multiples of 4)", list[i].n, list[i].plane);
      batch.s[i] = list[i];
      blocks += static_cast<unsigned>((list[i].n / 4 + 255) / 256);
    }
    batch.end[i] = blocks;
  }
  LaunchScope scope(stream, "sum_planes");
  return launch_kernel(stream, sum_planes_kernel, blocks, 256, 0, batch);
}

int launch_split_planes(cudaStream_t stream, const float* x, __nv_bfloat16* parts, long long plane, long long n) {
  KFB_CHECK_ARG(n % 4 == 0 && plane % 4 == 0, "split_planes: %lld elements, planes %lld apart (multiples of 4)", n, plane);
  LaunchScope scope(stream, "split_planes");
  return launch_kernel(stream, split_planes_kernel, static_cast<unsigned>((n / 4 + 255) / 256), 256, 0, x, parts, plane, n);
}

}  // namespace kfb
