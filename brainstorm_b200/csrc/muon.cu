// Momentum whose update is orthogonalised by Newton-Schulz products, for stacks of equally shaped
// matrices:
//
//   m = beta m + g;   u = g + beta m (Nesterov) or m;   X = u / (|u|_F + 1e-7)
//   `steps` times:    A = X X^T;  X = a X + (b A + c A A) X        (a, b, c) = (3.4445, -4.7750, 2.0315)
//   update = X;       p = (1 - rate * decay) p - rate X
//
// The iteration runs on X or X^T, whichever has no more rows than columns.
#include <algorithm>

#include "common.cuh"

namespace b200 {
int gemm_tc(int transa, int transb, int64_t M, int64_t N, int64_t K, const float* a, int64_t lda, const float* b, int64_t ldb, float* c,
            int64_t ldc, int accumulate);
int gemm_simt(int transa, int transb, int64_t M, int64_t N, int64_t K, const float* a, int64_t lda, const float* b, int64_t ldb, float* c,
              int64_t ldc, int accumulate);

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int MU_NORM_BLOCKS = 128;      // per matrix

// momentum update and, per block, the sum of squares of the direction (64 bits: no overflow, no rounding to speak of)
__global__ void __launch_bounds__(256) muon_momentum_kernel(const float* grad, float* momentum, int64_t size, float beta, int nesterov,
                                                            double* partial) {
  __shared__ double red[8];
  const float* g = grad + blockIdx.y * size;
  float* m = momentum + blockIdx.y * size;
  double s = 0.;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    const float gi = g[i], mi = beta * m[i] + gi;
    m[i] = mi;
    const float u = nesterov ? gi + beta * mi : mi;
    s += (double)u * u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.;
    for (int w = 0; w < 8; ++w) t += red[w];
    partial[blockIdx.y * gridDim.x + blockIdx.x] = t;
  }
}

__device__ __forceinline__ float muon_inverse_norm(const double* partial, int count, double* red) {
  double s = 0.;
  for (int i = threadIdx.x; i < count; i += blockDim.x) s += partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  double t = 0.;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return (float)(1. / (sqrt(t) + 1e-7));
}

// X = u / |u|, X^T when tall
__global__ void __launch_bounds__(256) muon_start_kernel(const float* grad, const float* momentum, int rows, int cols, float beta, int nesterov,
                                                         const double* partial, int partials, int tall, float* X) {
  __shared__ double red[8];
  __shared__ float tile[32][33];
  const int64_t size = (int64_t)rows * cols;
  const float* g = grad + blockIdx.z * size;
  const float* m = momentum + blockIdx.z * size;
  float* x = X + blockIdx.z * size;
  const float inv = muon_inverse_norm(partial + blockIdx.z * partials, partials, red);
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int y = ty; y < 32; y += 8) {
    const int r = r0 + y, c = c0 + tx;
    if (r < rows && c < cols) {
      const int64_t i = (int64_t)r * cols + c;
      const float u = nesterov ? g[i] + beta * m[i] : m[i];
      if (tall) tile[y][tx] = u * inv;
      else x[i] = u * inv;
    }
  }
  if (!tall) return;
  __syncthreads();
  for (int y = ty; y < 32; y += 8) {
    const int c = c0 + y, r = r0 + tx;
    if (r < rows && c < cols) x[(int64_t)c * rows + r] = tile[tx][y];
  }
}

__global__ void __launch_bounds__(256) muon_combine_kernel(const float* a, const float* aa, float* out, int64_t n, float fa, float faa) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = fa * a[i] + faa * aa[i];
}

// update = X (or its transpose), p = keep * p - rate * X
__global__ void __launch_bounds__(256) muon_apply_kernel(const float* X, float* update, float* param, int rows, int cols, int tall, float keep,
                                                         float rate) {
  __shared__ float tile[32][33];
  const int64_t size = (int64_t)rows * cols;
  const float* x = X + blockIdx.z * size;
  float* u = update + blockIdx.z * size;
  float* p = param + blockIdx.z * size;
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  if (tall) {
    for (int y = ty; y < 32; y += 8) {
      const int c = c0 + y, r = r0 + tx;
      if (r < rows && c < cols) tile[tx][y] = x[(int64_t)c * rows + r];
    }
    __syncthreads();
  }
  for (int y = ty; y < 32; y += 8) {
    const int r = r0 + y, c = c0 + tx;
    if (r < rows && c < cols) {
      const int64_t i = (int64_t)r * cols + c;
      const float v = tall ? tile[y][tx] : x[i];
      u[i] = v;
      p[i] = keep * p[i] - rate * v;
    }
  }
}

static int muon_gemm(int transb, int64_t M, int64_t N, int64_t K, const float* a, const float* b, float* c) {
  const int64_t ldb = transb ? K : N;
  const int rc = gemm_tc(0, transb, M, N, K, a, K, b, ldb, c, N, 0);
  return rc != B200_ERR_UNSUPPORTED ? rc : gemm_simt(0, transb, M, N, K, a, K, b, ldb, c, N, 0);
}

}  // namespace b200

using namespace b200;

B200_API int64_t b200_muon_scratch_floats(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  const int64_t m = std::min(rows, cols);
  return 2 * batch * rows * cols + 3 * m * m + 2 * batch * MU_NORM_BLOCKS + 16;
}

B200_API int b200_muon_update(float* param, const float* grad, float* momentum, float* update, int64_t batch, int64_t rows, int64_t cols,
                              float learning_rate, float beta, int nesterov, float weight_decay, int steps, float* scratch,
                              int64_t scratch_floats) {
  if (int rc = require_ready()) return rc;
  B200_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "negative extent");
  B200_REQUIRE(steps >= 0 && steps <= 100, "muon: %d steps", steps);
  if (batch == 0 || rows == 0 || cols == 0) return B200_OK;
  B200_REQUIRE(rows < (1 << 20) && cols < (1 << 20) && batch < 65536, "muon: extent too large");
  B200_REQUIRE(param && grad && momentum && update && scratch, "muon: NULL operand");
  B200_REQUIRE(scratch_floats >= b200_muon_scratch_floats(batch, rows, cols) && ((uintptr_t)scratch & 15) == 0, "muon: scratch too small");
  const cudaStream_t st = state().stream;
  const int tall = rows > cols;
  const int64_t m = tall ? cols : rows, n = tall ? rows : cols, size = m * n;
  double* partial = (double*)scratch;
  float* X = scratch + 2 * ((batch * MU_NORM_BLOCKS + 1) & ~(int64_t)1);
  float* Y = X + batch * size;
  float* A = Y + batch * size;
  float* AA = A + m * m;
  const unsigned nb = (unsigned)std::min<int64_t>(MU_NORM_BLOCKS, ceil_div(size, 1024));
  muon_momentum_kernel<<<dim3(nb, (unsigned)batch), 256, 0, st>>>(grad, momentum, size, beta, nesterov, partial);
  B200_LAUNCH_CHECK();
  const dim3 tiles((unsigned)ceil_div(cols, 32), (unsigned)ceil_div(rows, 32), (unsigned)batch);
  muon_start_kernel<<<tiles, 256, 0, st>>>(grad, momentum, (int)rows, (int)cols, beta, nesterov, partial, (int)nb, tall, X);
  B200_LAUNCH_CHECK();
  const unsigned eb = (unsigned)std::min<int64_t>(ceil_div(std::max(size, m * m), 256), (int64_t)state().sm_count * 8);
  float *from = X, *to = Y;
  for (int i = 0; i < steps; ++i) {
    for (int64_t b = 0; b < batch; ++b) {
      const float* x = from + b * size;
      float* y = to + b * size;
      if (int rc = muon_gemm(1, m, m, n, x, x, A)) return rc;
      if (int rc = muon_gemm(0, m, m, m, A, A, AA)) return rc;
      muon_combine_kernel<<<eb, 256, 0, st>>>(A, AA, A, m * m, NS_B, NS_C);
      B200_LAUNCH_CHECK();
      if (int rc = muon_gemm(0, m, n, m, A, x, y)) return rc;
      muon_combine_kernel<<<eb, 256, 0, st>>>(x, y, y, size, NS_A, 1.f);
      B200_LAUNCH_CHECK();
    }
    std::swap(from, to);
  }
  muon_apply_kernel<<<tiles, 256, 0, st>>>(from, update, param, (int)rows, (int)cols, tall, 1.f - learning_rate * weight_decay, learning_rate);
  B200_LAUNCH_CHECK();
  return B200_OK;
}
