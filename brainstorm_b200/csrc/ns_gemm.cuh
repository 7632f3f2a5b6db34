// Products of matrices that are stored as two half-precision planes (ns_gemm.cu).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

// A matrix (or a stack of them) as hi and lo planes: value = (hi + lo) / NS_SCALE.  Plane p of matrix b
// starts at (p * batch + b) * rows * ld; ld is a multiple of 8.
struct NsMatrix {
  __half* data;
  int rows, cols, ld;
};
constexpr float NS_SCALE = 4096.f;

// out = alpha * a b^T + beta * add, for each matrix of the stack; a is (M, K), b is (N, K), both with K along
// the rows.  symmetric: the product is known to be symmetric; one triangle is computed and stored twice.
// out_t, if given, receives the transpose (N, M).  add may be NULL, out may be NULL when out_t is given.
int ns_gemm(const NsMatrix& a, const NsMatrix& b, const NsMatrix* add, const NsMatrix* out, const NsMatrix* out_t, int batch, float alpha,
            float beta, bool symmetric);
}  // namespace b200
