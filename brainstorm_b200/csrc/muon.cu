// Momentum whose update is orthogonalised by Newton-Schulz products, for stacks of equally shaped
// matrices:
//
//   m = beta m + g;   u = g + beta m (Nesterov) or m;   X = u / (|u|_F + 1e-7)
//   `steps` times:    A = X X^T;  X = a X + (b A + c A A) X        (a, b, c) = (3.4445, -4.7750, 2.0315)
//   update = X;       p = (1 - rate * decay) p - rate X
//
// The iteration multiplies from the shorter side: with rows > cols, A = X^T X and X = X P.  P = a I + b A + c A A is
// computed as c D D + (a - b^2 / 4c) I with D = A + b / 2c I: three plain products a step, whose only addition is
// to a diagonal.
//
// Bound: the products (ns_gemm.cu).  4096 x 4096 takes 3.9 ms, of which they are 3.75 at 366 TFLOP/s of fp32 accuracy
// (1100 of half precision, at the clocks that the power limit leaves); four of 1000 x 1000 0.40 ms, half of it the first
// loads and the epilogues of fifteen products that each fill the GPU once; 205 x 256 92 us in one launch.
#include <algorithm>

#include "common.cuh"
#include "ns_gemm.cuh"

namespace b200 {

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int MU_NORM_BLOCKS = 512;      // at most, per matrix

// momentum update and, per block, the sum of squares of the direction (64 bits: no overflow, no rounding to speak of)
template <bool VEC>
__global__ void __launch_bounds__(256) muon_momentum_kernel(const float* grad, float* momentum, int64_t size, float beta, int nesterov,
                                                            double* partial) {
  __shared__ double red[8];
  const float* g = grad + blockIdx.y * size;
  float* m = momentum + blockIdx.y * size;
  double s = 0.;
  auto next = [&](float gi, float mi) {
    mi = beta * mi + gi;
    const double u = nesterov ? gi + beta * mi : mi;
    s += u * u;
    return mi;
  };
  const int64_t step = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (VEC) {
#pragma unroll 2
    for (int64_t i = first; i < size / 4; i += step) {
      const float4 a = reinterpret_cast<const float4*>(g)[i];
      float4 b = reinterpret_cast<float4*>(m)[i];
      b.x = next(a.x, b.x);
      b.y = next(a.y, b.y);
      b.z = next(a.z, b.z);
      b.w = next(a.w, b.w);
      reinterpret_cast<float4*>(m)[i] = b;
    }
  } else {
#pragma unroll 4
    for (int64_t i = first; i < size; i += step) m[i] = next(g[i], m[i]);
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

// The factor that makes planes of u / (|u| + 1e-7).  Formed in 64 bits: the inverse of a norm above 2^126 alone would lose bits in 32.
__device__ __forceinline__ float muon_plane_factor(const double* partial, int count, double* red) {
  double s = 0.;
  for (int i = threadIdx.x; i < count; i += blockDim.x) s += partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  double t = 0.;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return (float)((double)NS_SCALE / (sqrt(t) + 1e-7));
}

__device__ __forceinline__ void muon_split(float x, float y, __half2& hi, __half2& lo) {
  hi = __floats2half2_rn(x, y);
  const float2 f = __half22float2(hi);
  lo = __floats2half2_rn(x - f.x, y - f.y);
}

// X = u / |u| as planes, two values a thread at a time: block column x, rows y, matrix z.
__global__ void __launch_bounds__(256) muon_start_kernel(const float* grad, const float* momentum, float beta, int nesterov, const double* partial,
                                                         int partials, NsMatrix X) {
  __shared__ double red[8];
  const int64_t size = (int64_t)X.rows * X.cols, plane = (int64_t)gridDim.z * X.rows * X.ld;
  const float* g = grad + blockIdx.z * size;
  const float* m = momentum + blockIdx.z * size;
  __half* s = X.data + (int64_t)blockIdx.z * X.rows * X.ld;
  const int c = (blockIdx.x * 32 + (threadIdx.x & 31)) * 2, r0 = blockIdx.y * 64 + (threadIdx.x >> 5);
  float2 gv[8], mv[8];
#pragma unroll
  for (int y = 0; y < 8; ++y) {
    const int r = r0 + 8 * y;
    const int64_t i = (int64_t)r * X.cols + c;
    gv[y] = mv[y] = make_float2(0.f, 0.f);
    if (r < X.rows && c < X.cols) {
      gv[y].x = g[i];
      mv[y].x = m[i];
      if (c + 1 < X.cols) {
        gv[y].y = g[i + 1];
        mv[y].y = m[i + 1];
      }
    }
  }
  const float inv = muon_plane_factor(partial + blockIdx.z * partials, partials, red);
  __half2 hi, lo;
#pragma unroll
  for (int y = 0; y < 8; ++y) {
    const int r = r0 + 8 * y;
    if (r < X.rows && c < X.cols) {        // a pair may reach into the padding of the row
      muon_split((nesterov ? gv[y].x + beta * mv[y].x : mv[y].x) * inv, (nesterov ? gv[y].y + beta * mv[y].y : mv[y].y) * inv, hi, lo);
      *reinterpret_cast<__half2*>(s + (int64_t)r * X.ld + c) = hi;
      *reinterpret_cast<__half2*>(s + plane + (int64_t)r * X.ld + c) = lo;
    }
  }
}

// update = X, p = keep * p - rate * X.  VEC: rows are multiples of 8 values and
// all arrays start on 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(256) muon_apply_kernel(NsMatrix X, float* update, float* param, float keep, float rate) {
  const int64_t size = (int64_t)X.rows * X.cols, plane = (int64_t)gridDim.y * X.rows * X.ld;
  const __half* x = X.data + (int64_t)blockIdx.y * X.rows * X.ld;
  float* u = update + blockIdx.y * size;
  float* p = param + blockIdx.y * size;
  const int64_t step = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (VEC) {
    for (int64_t i = first; i < size / 8; i += step) {
      const uint4 h = reinterpret_cast<const uint4*>(x)[i], l = reinterpret_cast<const uint4*>(x + plane)[i];
      float4 a = reinterpret_cast<float4*>(p)[2 * i], b = reinterpret_cast<float4*>(p)[2 * i + 1];
      auto join = [](uint32_t hw, uint32_t lw) {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&hw)), e = __half22float2(*reinterpret_cast<__half2*>(&lw));
        return make_float2((f.x + e.x) * (1.f / NS_SCALE), (f.y + e.y) * (1.f / NS_SCALE));
      };
      const float2 v0 = join(h.x, l.x), v1 = join(h.y, l.y), v2 = join(h.z, l.z), v3 = join(h.w, l.w);
      reinterpret_cast<float4*>(u)[2 * i] = make_float4(v0.x, v0.y, v1.x, v1.y);
      reinterpret_cast<float4*>(u)[2 * i + 1] = make_float4(v2.x, v2.y, v3.x, v3.y);
      a = make_float4(keep * a.x - rate * v0.x, keep * a.y - rate * v0.y, keep * a.z - rate * v1.x, keep * a.w - rate * v1.y);
      b = make_float4(keep * b.x - rate * v2.x, keep * b.y - rate * v2.y, keep * b.z - rate * v3.x, keep * b.w - rate * v3.y);
      reinterpret_cast<float4*>(p)[2 * i] = a;
      reinterpret_cast<float4*>(p)[2 * i + 1] = b;
    }
  } else {
    for (int64_t i = first; i < size; i += step) {
      const int64_t at = i + i / X.cols * (X.ld - X.cols);
      const float v = (__half2float(x[at]) + __half2float(x[at + plane])) * (1.f / NS_SCALE);
      u[i] = v;
      p[i] = keep * p[i] - rate * v;
    }
  }
}

static int64_t muon_pitch(int64_t n) { return (n + 7) & ~(int64_t)7; }
// Planes of a (rows, cols) stack, in floats, a multiple of 128 bytes.
static int64_t muon_planes(int64_t batch, int64_t rows, int64_t cols) { return (batch * rows * muon_pitch(cols) + 31) & ~(int64_t)31; }

}  // namespace b200

using namespace b200;

B200_API int64_t b200_muon_scratch_floats(int64_t batch, int64_t rows, int64_t cols) {
  if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
  const int64_t m = std::min(rows, cols);
  return 2 * muon_planes(batch, rows, cols) + 2 * muon_planes(batch, m, m) + 2 * batch * MU_NORM_BLOCKS + 64;
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
  const int64_t m = std::min(rows, cols), size = rows * cols;
  float* at = (float*)(((uintptr_t)scratch + 127) & ~(uintptr_t)127);      // TMA wants 16 bytes, whole lines are better
  auto planes = [&](int64_t r, int64_t c) {
    NsMatrix x = {(__half*)at, (int)r, (int)c, (int)muon_pitch(c), 0};
    at += muon_planes(batch, r, c);
    return x;
  };
  NsMatrix X[2] = {planes(rows, cols), planes(rows, cols)}, D = planes(m, m), P = planes(m, m);
  double* partial = (double*)at;
  // whole lines for each matrix of the stack, or single values
  const bool vec = size % 4 == 0 && aligned16(grad) && aligned16(momentum);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(MU_NORM_BLOCKS, (int64_t)state().sm_count * 8 / batch));
  const unsigned nb = (unsigned)std::min<int64_t>(want, ceil_div(size, 1024));
  (vec ? muon_momentum_kernel<true> : muon_momentum_kernel<false>)<<<dim3(nb, (unsigned)batch), 256, 0, st>>>(grad, momentum, size, beta, nesterov, partial);
  B200_LAUNCH_CHECK();
  const dim3 tiles((unsigned)ceil_div(cols, 64), (unsigned)ceil_div(rows, 64), (unsigned)batch);
  muon_start_kernel<<<tiles, 256, 0, st>>>(grad, momentum, beta, nesterov, partial, (int)nb, X[0]);
  B200_LAUNCH_CHECK();
  constexpr float d_diagonal = NS_B / (2.f * NS_C), p_diagonal = NS_A - NS_B * NS_B / (4.f * NS_C);
  int now = steps & 1;
  if (steps > 0 && ns_chain_fits(rows, cols, batch)) {
    if (int rc = ns_chain(X, D, P, tall, (int)batch, steps, d_diagonal, NS_C, p_diagonal)) return rc;
  } else {
    for (int i = 0; i < steps; ++i) {
      const NsMatrix& x = X[i & 1];
      NsMatrix* y = &X[~i & 1];
      if (int rc = ns_gemm(x, tall, x, tall, &D, (int)batch, 1.f, d_diagonal, true)) return rc;       // from X X^T, or X^T X
      if (int rc = ns_gemm(D, false, D, false, &P, (int)batch, NS_C, p_diagonal, true)) return rc;
      const int rc = tall ? ns_gemm(x, false, P, false, y, (int)batch, 1.f, 0.f, false)              // X P, P symmetric
                          : ns_gemm(P, false, x, true, y, (int)batch, 1.f, 0.f, false);              // P X
      if (rc) return rc;
    }
  }
  const unsigned eb = (unsigned)std::min<int64_t>(ceil_div(size, 2048), (int64_t)state().sm_count * 8);
  const bool whole = cols % 8 == 0 && aligned16(update) && aligned16(param);
  (whole ? muon_apply_kernel<true> : muon_apply_kernel<false>)<<<dim3(eb, (unsigned)batch), 256, 0, st>>>(
      X[now], update, param, 1.f - learning_rate * weight_decay, learning_rate);
  B200_LAUNCH_CHECK();
  return B200_OK;
}
