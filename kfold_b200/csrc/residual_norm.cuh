// What lies between two blocks of a residual stream: how its rows are walked (residual_norm.cu, residual_norm_grad.cu).
//
// Row (group, sample, token) of the stream has the gates of row (group, token).  A team takes the samples that share a gate row one after the other, so that
// gates are read and their exponentials computed once for all of them; where gate rows are few, their samples are cut into pieces.
// Rows come through a ring in shared memory, slots of 16 bytes a thread: a thread copies the pieces that it will work on itself, several rows
// ahead, and needs neither registers nor barriers for them.  (The same loads into registers one row ahead, at the one block of 256 threads an SM that 200
// registers allow, moved 2.3 TB/s.)
#pragma once
#include "row_teams.cuh"

namespace kfb {

enum RowNorm : int { kNoNorm = 0, kAffineNorm = 1, kAdaptiveNorm = 2 };

// What a kernel is made for: gates that samples share (of the output, the norm or both), gates of a row's own with a norm without them, and with the adaptive
// one.  Each keeps other things in registers from row to row.
enum RowGates : int { kSharedGates = 0, kOwnGates = 1, kOwnAdaptive = 2 };

constexpr int kRowThreads = 128;

struct RowPlan {
  unsigned gate_rows, l;     // l tokens a group
  int samples;
  int chunks, chunk;         // pieces of a gate row's samples, and how many samples a piece has (the last may have fewer)
  unsigned units, sets;      // pieces; and as warps take them
};

// The rows of one team of a warp.  OWN: every row has gates of its own.
template <int LANES, bool OWN>
struct Walk {
  unsigned set, row = 0, unit = 0;
  int at = 0, left = 0;      // samples that the warp has taken of this piece; that are left to this team
  __device__ __forceinline__ void enter(const RowPlan& p, int team) {
    unit = set * (32 / LANES) + team;
    const bool there = unit < p.units;
    if (OWN) {
      row = there ? unit : 0;
      left = there ? 1 : 0;
    } else {
      const unsigned u = there ? unit : 0, gate = u / p.chunks, first = u % p.chunks * p.chunk;
      left = there ? min(p.chunk, p.samples - static_cast<int>(first)) : 0;
      row = (gate / p.l * p.samples + first) * p.l + gate % p.l;
    }
  }
  __device__ __forceinline__ void next(const RowPlan& p, int team, unsigned step) {
    if (OWN || ++at == p.chunk) {
      at = 0;
      set += step;
      if (set < p.sets) enter(p, team);
    } else {
      --left;
      row += p.l;
    }
  }
  __device__ __forceinline__ unsigned gate_row(const RowPlan& p) const { return OWN ? row : unit < p.units ? unit / p.chunks : 0; }
};

// A plan for `teams` teams at work at once, `in_warp` of them in a warp: pieces that the teams finish together.  The cost of a round is its samples and, for the
// gates and the sums, about two more; where a second kernel has to join pieces of `unit_bytes`, written and read, its launch costs 1.3 and seven megabytes one
// (the gradient of 301 gate rows of five samples of 768 channels: whole 12.9 us, cut 14.4; of 64: 12.4 and 8.9).
// Never more than two pieces a team.
inline RowPlan row_plan(long long rows, int samples, int l, long long teams, int in_warp, int unit_bytes) {
  RowPlan p = {};
  p.gate_rows = static_cast<unsigned>(rows / samples);
  p.l = static_cast<unsigned>(l);
  p.samples = samples;
  p.chunks = 1;
  double best = 0.;
  for (int k = 1; k <= samples; k += k < 64 ? 1 : k / 32) {      // (thousands of samples are not gone through one by one)
    const long long units = static_cast<long long>(p.gate_rows) * k;
    if (k > 1 && units > 2 * teams) break;
    const double join = k > 1 && unit_bytes > 0 ? 1.3 + 1.5e-7 * units * unit_bytes : 0.;
    const double cost = static_cast<double>((units + teams - 1) / teams * ((samples + k - 1) / k + 2)) + join;
    if (k == 1 || cost < best) {
      best = cost;
      p.chunks = k;
    }
  }
  p.chunk = (samples + p.chunks - 1) / p.chunks;
  p.chunks = (samples + p.chunk - 1) / p.chunk;
  p.units = p.gate_rows * p.chunks;
  p.sets = (p.units + in_warp - 1) / in_warp;
  return p;
}

// Sums of K values over a team's lanes, the same in all of them.
template <int LANES, int K>
__device__ __forceinline__ void team_sum(float (&v)[K]) {
#pragma unroll
  for (int m = LANES / 2; m > 0; m >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
}

// The ring.  Bytes that an SM's blocks have for it, and rows on their way for a team, the one in work among them: 2 to 4, as many as leave `blocks`
// of 128 threads an SM their place.  (Gates of a row's own leave registers for three, and their exponentials want the warps more than a third row on its way.)
constexpr int kMostRing = 216 * 1024;
constexpr int ring_depth(int row_bytes, int blocks) {      // of a thread and row
  const int d = kMostRing / blocks / kRowThreads / row_bytes;
  return d < 2 ? 2 : d > 4 ? 4 : d;
}
// Slot `s` of stage `q` of this thread: ring + ((q * slots + s) * kRowThreads + thread) * 16 bytes; piece p of a tensor p * (16-byte words of a piece) slots on.
// `from`: this lane's first piece of a row, the others STEP elements apart; there: P flags, which pieces there are.
template <typename T, int P, int STEP>
__device__ __forceinline__ void ring_copy(uint32_t slot, const T* from, const bool (&there)[P]) {
  constexpr int kWords = sizeof(T) / 2;
#pragma unroll
  for (int q = 0; q < P; ++q)
#pragma unroll
    for (int i = 0; i < kWords; ++i) copy_async<16>(slot + (q * kWords + i) * kRowThreads * 16, reinterpret_cast<const uint4*>(from + q * STEP) + i, there[q]);
}
// Rows in 8 bits: the bytes, and where `words` says so the words of exponents that the pieces' lie in (`exponents`: a row's).
template <int P, int STEP>
__device__ __forceinline__ void ring_copy8(uint32_t slot, const uint8_t* from, const uint8_t* exponents, int channel, bool words, const bool (&there)[P]) {
#pragma unroll
  for (int q = 0; q < P; ++q) {
    copy_async<8>(slot + q * kRowThreads * 16, from + q * STEP, there[q]);
    if (words) copy_async<4>(slot + q * kRowThreads * 16 + 8, exponents + ((channel + q * STEP) / kGroup8 & ~3), there[q]);
  }
}
// Rows of other widths or addresses are read as they lie; a warp asks for the next one's lines ahead.
template <typename T>
__device__ __forceinline__ void prefetch_row(const T* row, int c, int lane) {
  for (int i = lane * (128 / static_cast<int>(sizeof(T))); i < c; i += 32 * (128 / static_cast<int>(sizeof(T))))
    asm volatile("prefetch.global.L2 [%0];" ::"l"(row + i));
}

template <typename T>
__device__ __forceinline__ Pairs ring_take(const uint4* slot) {
  if constexpr (sizeof(T) == 2) return of_bf16(slot[0]);
  else return of_f32(slot[0], slot[kRowThreads]);
}

// The kernels' shapes: lanes of a team and pieces of a lane, two at least where there are, for fewer instructions a row (the gradient of 384 x 384 rows of 128 channels 32 us,
// 41 with 16 lanes of one).  CALL(LANES, P, VEC) for c channels.
#define KFB_ROW_SHAPES(c, vec, CALL)                  \
  do {                                                \
    if (vec) {                                        \
      if ((c) <= 64) return CALL(8, 1, true);         \
      if ((c) <= 128) return CALL(8, 2, true);        \
      if ((c) <= 256) return CALL(16, 2, true);       \
      if ((c) <= 384) return CALL(16, 3, true);       \
      if ((c) <= 512) return CALL(32, 2, true);       \
      if ((c) <= 768) return CALL(32, 3, true);       \
      return CALL(32, 4, true);                       \
    }                                                 \
    if ((c) <= 256) return CALL(32, 1, false);        \
    if ((c) <= 512) return CALL(32, 2, false);        \
    return CALL(32, 4, false);                        \
  } while (0)

}  // namespace kfb
