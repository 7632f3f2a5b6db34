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
#include "ns_gemm.cuh"

namespace b200 {

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

// X = u / |u| and its transpose, as planes.  Tiles of 32 x 32 through shared memory; block z: matrix.
// straight receives u's own orientation, turned the transposed one.
__global__ void __launch_bounds__(256) muon_start_kernel(const float* grad, const float* momentum, int rows, int cols, float beta, int nesterov,
                                                         const double* partial, int partials, NsMatrix straight, NsMatrix turned) {
  __shared__ double red[8];
  __shared__ float tile[32][33];
  const int64_t size = (int64_t)rows * cols;
  const float* g = grad + blockIdx.z * size;
  const float* m = momentum + blockIdx.z * size;
  const float inv = NS_SCALE * muon_inverse_norm(partial + blockIdx.z * partials, partials, red);
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t plane = (int64_t)gridDim.z * straight.rows * straight.ld, plane_t = (int64_t)gridDim.z * turned.rows * turned.ld;
  __half* s = straight.data + (int64_t)blockIdx.z * straight.rows * straight.ld;
  __half* t = turned.data + (int64_t)blockIdx.z * turned.rows * turned.ld;
  auto put = [](__half* at, int64_t plane, float x) {
    const __half h = __float2half_rn(x);
    at[0] = h;
    at[plane] = __float2half_rn(x - __half2float(h));
  };
#pragma unroll
  for (int y = ty; y < 32; y += 8) {
    const int r = r0 + y, c = c0 + tx;
    float x = 0.f;
    if (r < rows && c < cols) {
      const int64_t i = (int64_t)r * cols + c;
      x = (nesterov ? g[i] + beta * m[i] : m[i]) * inv;
      put(s + (int64_t)r * straight.ld + c, plane, x);
    }
    tile[y][tx] = x;
  }
  __syncthreads();
#pragma unroll
  for (int y = ty; y < 32; y += 8) {
    const int c = c0 + y, r = r0 + tx;
    if (r < rows && c < cols) put(t + (int64_t)c * turned.ld + r, plane_t, tile[tx][y]);
  }
}

// update = X, p = keep * p - rate * X, X in the parameters' own orientation
__global__ void __launch_bounds__(256) muon_apply_kernel(NsMatrix X, float* update, float* param, float keep, float rate) {
  const int64_t size = (int64_t)X.rows * X.cols, plane = (int64_t)gridDim.y * X.rows * X.ld;
  const __half* x = X.data + (int64_t)blockIdx.y * X.rows * X.ld;
  float* u = update + blockIdx.y * size;
  float* p = param + blockIdx.y * size;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    const int64_t r = X.ld == X.cols ? 0 : i / X.cols;
    const int64_t at = i + r * (X.ld - X.cols);
    const float v = (__half2float(x[at]) + __half2float(x[at + plane])) * (1.f / NS_SCALE);
    u[i] = v;
    p[i] = keep * p[i] - rate * v;
  }
}

static int64_t muon_pitch(int64_t n) { return (n + 7) & ~(int64_t)7; }
// Planes of a (rows, cols) stack, in floats, a multiple of 128 bytes.
static int64_t muon_planes(int64_t batch, int64_t rows, int64_t cols) { return (batch * rows * muon_pitch(cols) + 31) & ~(int64_t)31; }

}  // namespace b200

using namespace b200;

B200_API int64_t b200_muon_scratch_floats(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
  return 2 * muon_planes(batch, m, n) + 2 * muon_planes(batch, n, m) + 2 * muon_planes(batch, m, m) + 2 * batch * MU_NORM_BLOCKS + 64;
}

B200_API int b200_muon_update(float* param, const float* grad, float* momentum, float* update, int64_t batch, int64_t rows, int64_t cols,
                              float learning_rate, float beta, int nesterov, float weight_decay, int steps, float* scratch,
                              int64_t scratch_floats) {
  if (int rc = require_ready()) return rc;
  B200_REQUIRE(batch >= 0 && rows >= 0 && cols >= 0, "negative extent");
  B200_REQUIRE(steps >= 0 && steps <= 100, "muon: %d steps", steps);
  if (batch == 0 || rows == 0 || cols == 0) return B200_OK;
  B200_REQUIRE(rows < (1 << 20) && cols < (1 << 20) && batch < 32768, "muon: extent too large");
  B200_REQUIRE(param && grad && momentum && update && scratch, "muon: NULL operand");
  B200_REQUIRE(scratch_floats >= b200_muon_scratch_floats(batch, rows, cols) && ((uintptr_t)scratch & 15) == 0, "muon: scratch too small or misaligned");
  const cudaStream_t st = state().stream;
  const bool tall = rows > cols;
  const int64_t m = tall ? cols : rows, n = tall ? rows : cols, size = m * n;
  float* at = (float*)(((uintptr_t)scratch + 127) & ~(uintptr_t)127);      // TMA wants 16 bytes, whole lines are better
  auto planes = [&](int64_t r, int64_t c) {
    NsMatrix x = {(__half*)at, (int)r, (int)c, (int)muon_pitch(c)};
    at += muon_planes(batch, r, c);
    return x;
  };
  NsMatrix X[2] = {planes(m, n), planes(m, n)}, Y[2] = {planes(n, m), planes(n, m)}, A = planes(m, m), B = planes(m, m);      // Y = X^T
  double* partial = (double*)at;
  const unsigned nb = (unsigned)std::min<int64_t>(MU_NORM_BLOCKS, ceil_div(size, 1024));
  muon_momentum_kernel<<<dim3(nb, (unsigned)batch), 256, 0, st>>>(grad, momentum, size, beta, nesterov, partial);
  B200_LAUNCH_CHECK();
  const dim3 tiles((unsigned)ceil_div(cols, 32), (unsigned)ceil_div(rows, 32), (unsigned)batch);
  muon_start_kernel<<<tiles, 256, 0, st>>>(grad, momentum, (int)rows, (int)cols, beta, nesterov, partial, (int)nb, tall ? Y[0] : X[0], tall ? X[0] : Y[0]);
  B200_LAUNCH_CHECK();
  int now = 0;
  for (int i = 0; i < steps; ++i, now ^= 1) {
    const bool last = i == steps - 1;
    if (int rc = ns_gemm(X[now], X[now], nullptr, &A, &A, (int)batch, 1.f, 0.f, true)) return rc;
    if (int rc = ns_gemm(A, A, &A, &B, &B, (int)batch, NS_C, NS_B, true)) return rc;
    // the last result is only needed as the parameters lie
    if (int rc = ns_gemm(B, Y[now], &X[now], last && tall ? nullptr : &X[now ^ 1], last && !tall ? nullptr : &Y[now ^ 1], (int)batch, 1.f, NS_A, false))
      return rc;
  }
  const unsigned eb = (unsigned)std::min<int64_t>(ceil_div(size, 1024), (int64_t)state().sm_count * 8);
  muon_apply_kernel<<<dim3(eb, (unsigned)batch), 256, 0, st>>>(tall ? Y[now] : X[now], update, param, 1.f - learning_rate * weight_decay, learning_rate);
  B200_LAUNCH_CHECK();
  return B200_OK;
}
