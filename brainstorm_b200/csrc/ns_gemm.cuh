// Products of matrices that are stored as two half-precision planes (ns_gemm.cu).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

// A matrix (or a stack of them) as hi and lo planes: value = (hi + lo) / NS_SCALE.  Plane p of matrix b
// starts at (p * batch + b) * rows * ld; ld is a multiple of 8.  `upper`: the matrix is symmetric and only its
// blocks (i, j) of upper x upper with j >= i are stored (0: all of it).
struct NsMatrix {
  __half* data;
  int rows, cols, ld, upper;
};
constexpr float NS_SCALE = 4096.f;

// out = alpha * op(a) op(b)^T + diagonal * I, for each matrix of the stack; op(x) is x, (rows, K), or with _t the
// transpose of x, stored (K, rows).  symmetric: the product is known to be symmetric; only its upper blocks are
// computed, and out->upper is set.
int ns_gemm(const NsMatrix& a, bool a_t, const NsMatrix& b, bool b_t, NsMatrix* out, int batch, float alpha, float diagonal, bool symmetric);

// `steps` times D = X X^T + d_diagonal I (tall: X^T X), P = p_alpha D D + p_diagonal I, X = P X (tall: X P), from X[0]; step i
// ends in X[(i + 1) & 1].  One launch, for matrices that ns_chain_fits.
bool ns_chain_fits(int64_t rows, int64_t cols, int64_t batch);
int ns_chain(const NsMatrix* X, const NsMatrix& D, const NsMatrix& P, bool tall, int batch, int steps, float d_diagonal, float p_alpha, float p_diagonal);
}  // namespace b200
