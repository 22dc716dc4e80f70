// What lies between two blocks of a residual stream: how its rows are walked (residual_norm.cu, residual_norm_grad.cu).
//
// Row (group, sample, token) of the stream has the gates of row (group, token).  A team takes the samples that share a gate row one after the other, so that
// gates are read and their exponentials computed once for all of them; where gate rows are few, their samples are cut into pieces.
// Rows come through a ring in shared memory, a slot of 16 bytes a thread and tensor: a thread copies the pieces that it will work on itself, several rows
// ahead, and needs neither registers nor barriers for them.  (The same loads into registers one row ahead, at the one block of 256 threads an SM that 200
// registers allow, moved 2.3 TB/s.)
#pragma once
#include "row_teams.cuh"

namespace kfb {

enum RowNorm : int { kNoNorm = 0, kAffineNorm = 1, kAdaptiveNorm = 2 };

struct RowPlan {
  unsigned gate_rows, l;     // l tokens a group
  int samples;
  int chunks, chunk;         // pieces of a gate row's samples, and how many samples a piece has (the last may have fewer)
  unsigned units, sets;      // pieces; and as groups of lanes take them
};

// OWN: every row has gates of its own.
template <int LANES, bool OWN>
struct Walk {
  unsigned set, row = 0, unit = 0;
  int at = 0, left = 0;      // samples that the group has taken of this piece; that are left to this team
  __device__ __forceinline__ void enter(const RowPlan& p, int team) {
    unit = set * Teams<LANES>::kTeams + team;
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

// A plan for `teams` teams at work at once, kTeams of them in a group of lanes: pieces that the teams finish together.  The cost of a round is its
// samples and, for the gates and the sums, about two more.  Never more than two pieces a team.
inline RowPlan row_plan(long long rows, int samples, int l, long long teams, int teams_in_group) {
  RowPlan p = {};
  p.gate_rows = static_cast<unsigned>(rows / samples);
  p.l = static_cast<unsigned>(l);
  p.samples = samples;
  p.chunks = 1;
  long long best = -1;
  for (int k = 1; k <= samples; ++k) {
    const long long units = static_cast<long long>(p.gate_rows) * k, cost = (units + teams - 1) / teams * ((samples + k - 1) / k + 2);
    if (k > 1 && units > 2 * teams) break;
    if (best < 0 || cost < best) {
      best = cost;
      p.chunks = k;
    }
  }
  p.chunk = (samples + p.chunks - 1) / p.chunks;
  p.chunks = (samples + p.chunk - 1) / p.chunk;
  p.units = p.gate_rows * p.chunks;
  p.sets = (p.units + teams_in_group - 1) / teams_in_group;
  return p;
}

// The ring: slot `s` of stage `q` of this thread at ring[(q * slots + s) * threads], a piece of float32 in two neighbouring slots.
template <typename T, bool VEC>
__device__ __forceinline__ void ring_copy(uint4* slot, int stride, const T* from, bool there) {
#pragma unroll
  for (int i = 0; i < kPiece * static_cast<int>(sizeof(T)) / 16; ++i) copy_async16(slot + i * stride, reinterpret_cast<const uint4*>(from) + i, there);
}
__device__ __forceinline__ void ring_copy8(uint4* slot, const uint8_t* values, const uint8_t* words, bool there) {
  copy_async<8>(slot, values, there);
  copy_async<4>(reinterpret_cast<uint32_t*>(slot) + 2, words, there);
}

}  // namespace kfb
