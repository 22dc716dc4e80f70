// The hidden channels of a gated feed-forward, forward and for the gradient, in one kernel (feed_forward_hidden.cu).
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace kfb {

// bf16 rows.  dy == nullptr: h = silu(x Wa^T) (x Wb^T).  Otherwise also dab = [da, db] from dh = dy Wo (wo: (c, hidden) as it is stored).
// x, dy (rows, c), w_in (2 hidden, c), h (rows, hidden), dab (rows, 2 hidden).
bool ffn_hidden_ok(int c, int hidden);      // multiples of 64, and a device that holds a pair of CTAs
int launch_ffn_hidden(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, void* h, void* dab, int rows, int c,
                      int hidden);

// The same rows' dx (rows, c) in one kernel (feed_forward_rows.cu): 128 or 256 channels, hidden a multiple of 128.  h and dab as above, or both null
// where nobody wants them.
bool ffn_rows_ok(int c, int hidden);
int launch_ffn_rows(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, void* dx, void* h, void* dab, int rows,
                    int c, int hidden);

// The weights' gradients from x and dy alone (feed_forward_weights.cu): 128 channels, hidden a multiple of 64.  dw_in (2 hidden, c) and dw_out (c, hidden),
// either may be null: ffn_weights_planes float32 planes of each, to be added up.
bool ffn_weights_ok(int c, int hidden);
int ffn_weights_planes(long long rows, int hidden);
int launch_ffn_weights(cudaStream_t stream, const void* x, const void* dy, const void* w_in, const void* w_out, float* dw_in, float* dw_out, int rows,
                       int hidden);

// ... and from what was kept (feed_forward_sums.cu): 256 channels, hidden a multiple of 64.  `splits` planes (ffn_sums_planes; fewer where there are fewer
// blocks of 64 rows) are written, or added to.
bool ffn_sums_ok(int c, int hidden);
int ffn_sums_planes(long long rows, int hidden);
int launch_ffn_sums(cudaStream_t stream, const void* dab, const void* x, const void* h, const void* dy, float* dw_in, float* dw_out, int splits, int add,
                    int rows, int hidden);

}  // namespace kfb
