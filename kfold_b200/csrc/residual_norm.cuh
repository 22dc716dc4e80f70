// What lies between two blocks of a residual stream (residual_norm.cu, residual_norm_grad.cu).
#pragma once
#include <stdint.h>

namespace kfb {

enum RowNorm : int { kNoNorm = 0, kAffineNorm = 1, kAdaptiveNorm = 2 };

// Row (group, sample, token) of the stream has the gates of row (group, token): l tokens a group, `samples` entries that share.
struct RowShare {
  unsigned cond_rows, l;
  int samples;
  // the stream's row of a gate row's sample
  __device__ __forceinline__ unsigned row(unsigned cond, int sample) const {
    return samples == 1 ? cond : (cond / l * samples + sample) * l + cond % l;
  }
};

}  // namespace kfb
