// Products of bf16 matrices of either storage order on the tensor core (matmul.cu): the products of a backward pass, whose contraction
// runs over the rows of its operands as often as over their columns.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace kfb {

// An operand X(i, k), i = 0 ... extent - 1: stored [i][k] (by_k = 0) or [k][i] (by_k = 1), rows `ld` elements apart (a multiple of 8; the
// base 16-byte aligned).  plane: distance between its three bf16 parts in the fp32-accurate mode.
struct MatOperand {
  const void* ptr;
  long long ld;
  int by_k;
  long long plane;
};

// What becomes of a product z instead of being written as it is (a linear layer's tail, linear_tail.cuh); all products of a launch have one or none.
struct MatmulTail {
  int backward;          // 0: d = f(z + bias) + aux;  1: d = aux f'(z + bias), and its sums over rows
  int act;
  const float* bias;
  const void* aux;       // [m][ld_d], may be null in the forward direction
  int aux_fp32;
  int parts;             // 3: d is bf16 in three parts, plane_d apart; 1: bf16 or fp32 as out_fp32 says
  float* partial;        // backward, or null: [4 per 128 rows][n] sums of d before it is rounded
};

// D[m][n] = sum over k of A(m, k) B(n, k), accumulated in fp32.
struct MatmulArgs {
  MatOperand a, b;
  int m, n;
  long long k;
  void* d;               // [m][ld_d], bf16 or fp32
  long long ld_d;
  int out_fp32;
  int splits;            // fp32 D only: k in this many pieces, piece s into D + s * plane_d (none of them empty)
  long long plane_d;
  int accumulate;        // fp32 D only: add to what D holds
  int precise;           // operands are three bf16 parts each
  const MatmulTail* tail;
  int turns;             // fp32-accurate mode: accumulators that the large products' blocks of k go to in turn (matmul.cu), up to kMostTurns; 0 is one
};
static constexpr int kMostTurns = 3;
static constexpr int kMostMatmuls = 3;
// Up to kMostMatmuls products in one launch, all of them precise or none.
int launch_matmuls(cudaStream_t stream, const MatmulArgs* list, int count, const char* tag);
inline int launch_matmul(cudaStream_t stream, const MatmulArgs& p, const char* tag) { return launch_matmuls(stream, &p, 1, tag); }

// out[i] = sum over s of planes[s * plane + i], i < n, in the order of s; bf16 or fp32.  Up to kMostMatmuls of them in one launch.
struct PlaneSum {
  const float* planes;
  long long plane;
  int splits;
  void* out;
  int out_fp32;
  long long n;           // a multiple of 4, as plane is
};
int launch_sum_planes(cudaStream_t stream, const PlaneSum* list, int count);

// Three bf16 parts of n floats (a multiple of 4): parts[q * plane + i], x = x0 + x1 + x2.
int launch_split_planes(cudaStream_t stream, const float* x, __nv_bfloat16* parts, long long plane, long long n);

}  // namespace kfb
