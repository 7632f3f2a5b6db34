// Norms before and after a block, fused with the block's gate and residual scale.
//
//   n  = y * r_post * w_post          r_post = (mean(y^2) + eps)^(-1/2)      the norm after the block
//   x' = x + scale * act(gate) * n                                           gate, residual scale, residual
//   h  = x' * r_pre * w_pre           r_pre = (mean(x'^2) + eps)^(-1/2)      the norm before the next block
//
// One pass over the data in each direction: a row lives in the registers of its threads between the
// loads and the stores, both means are taken there, and nothing is read twice.  Backward, with
// x^ = x' r_pre, y^ = y r_post, e = dh w_pre, a = act(gate):
//
//   G  = dx' + r_pre (e - x^ mean(e x^))       dx = G          dw_pre = sum_rows dh x^
//   dgate = G scale n act'                                     dscale = sum_rows G a n
//   f  = G scale a w_post;  dy = r_post (f - y^ mean(f y^))    dw_post = sum_rows G scale a y^
//
// The column sums are kept per block in shared memory (a thread owns its columns, so there is nothing
// to synchronise), leave one row of partials per block, and are added in a fixed order by a second
// kernel: no atomics, the same bits every time.
//
// Bound: HBM where rows fill the vectors.  Forward moves 5 arrays, backward 8: 8192 x 4096 in 117 and 197 us, 5.7 and
// 5.5 TB/s.  Rows that start anywhere (3001 x 1537): 31 and 52 us, 3.0 and 2.9 TB/s, the latency of a row's two sums in the
// blocks that registers allow; the next row through shared memory instead of L2 gave 30 and 61.  Few rows: the
// latency of one (128 x 1000: 3.3 and 7.0 us).  Rows of 8193 to 16384 values hold 16 floats a thread on 1024 threads, whose 64
// registers are too few for a backward pass: 1500 x 16384 127 and 394 us (floors 75 and 120), 1500 x 16383, by single loads, 278 and 832.
// Added gradients read what was there: 8192 x 4096 294 us (floor 226), 3001 x 1537 67 (31), 1000000 x 32 809 (215).
#include <algorithm>
#include <initializer_list>
#include <utility>

#include "../../include/b200_handler.h"
#include "common.cuh"

namespace b200 {

constexpr int GN_MAX_WIDTH = 16384;

struct GatedNorm {
  const float *x, *y, *gate, *w_post, *scale, *w_pre;
  float *x_out, *h_out, *r_post, *r_pre;
  int64_t rows, ld_x, ld_y, ld_gate, ld_x_out, ld_h_out;
  int width, act;
  float eps;
};
struct GatedNormGrad {
  const float *x_out, *y, *gate, *w_post, *scale, *w_pre, *r_post, *r_pre, *dx_out, *dh;
  float *dx, *dy, *dgate, *partials;       // partials: one row of 3 * width sums (dw_post, dscale, dw_pre) per block
  int64_t rows, ld_x_out, ld_y, ld_gate, ld_dx_out, ld_dh, ld_dx, ld_dy, ld_dgate;
  int width, act, accumulate;
};

// x^(-1/2): the approximation (two units in the last place) and a Newton step, which 0 and infinity do not take.
__device__ __forceinline__ float gn_rsqrt(float x) {
  const float r = rsqrtf(x), e = fmaf(-x * r, r, 1.f);
  return e == e ? fmaf(0.5f * r, e, r) : r;
}
// The activations of the handler (0 sigmoid, 1 tanh, 2 rel, 3 el, 4 linear) and their derivatives as
// functions of the output.
__device__ __forceinline__ float gn_act(int act, float x) {
  switch (act) {
    case 0: return __fdividef(1.f, 1.f + expf(-x));      // two units in the last place; 0 for x < -87
    case 1: return tanhf(x);
    case 2: return x > 0.f ? x : (x == x ? 0.f : x);
    case 3: return x > 0.f ? x : expm1f(x);
    default: return x;
  }
}
__device__ __forceinline__ float gn_act_deriv(int act, float a) {
  switch (act) {
    case 0: return a * (1.f - a);
    case 1: return 1.f - a * a;
    case 2: return a > 0.f ? 1.f : 0.f;
    case 3: return a > 0.f ? 1.f : a + 1.f;
    default: return 1.f;
  }
}

// A row is held by G threads (a power of two, 32 .. 1024), E floats each.  MODE
//   GN_SINGLE: float number i * G + t of the row, one at a time;
//   GN_VEC:    float4 number i * G + t; all rows start on 16 bytes and hold a multiple of 4;
//   GN_SHIFT:  any width and start, all arrays alike: float4 number i * G + t counted from the 16-byte boundary at or
//              before the row, `off` floats (0 .. 3) ahead of it.  A thread meets rows of one `off` only (their distance is
//              a multiple of 4 rows), so its columns stay the same: column c of slot (i, j) is 4 (i G + t) + j - off.
enum { GN_SINGLE = 0, GN_VEC = 1, GN_SHIFT = 2 };
template <int MODE>
__device__ __forceinline__ int gn_column(int e, int G, int t, int off) {
  return MODE == GN_SINGLE ? e * G + t : 4 * ((e / 4) * G + t) + e % 4 - (MODE == GN_SHIFT ? off : 0);
}
template <int E, int MODE>
__device__ __forceinline__ void gn_load(float (&v)[E], const float* row, int width, int G, int t, int off) {
  if (MODE == GN_SINGLE) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e * G + t < width ? row[e * G + t] : 0.f;
    return;
  }
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const int c = gn_column<MODE>(4 * i, G, t, off);
    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
    if (MODE == GN_VEC ? c < width : c >= 0 && c + 4 <= width) {
      q = *reinterpret_cast<const float4*>(row + c);
    } else if (MODE == GN_SHIFT && c < width) {          // the ends of the row
      if (c >= 0) q.x = row[c];
      if (c + 1 >= 0 && c + 1 < width) q.y = row[c + 1];
      if (c + 2 >= 0 && c + 2 < width) q.z = row[c + 2];
      if (c + 3 >= 0 && c + 3 < width) q.w = row[c + 3];
    }
    v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
  }
}
template <int E, int MODE>
__device__ __forceinline__ void gn_store(const float (&v)[E], float* row, int width, int G, int t, int off) {
  if (MODE == GN_SINGLE) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e * G + t < width) row[e * G + t] = v[e];
    return;
  }
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const int c = gn_column<MODE>(4 * i, G, t, off);
    if (MODE == GN_VEC ? c < width : c >= 0 && c + 4 <= width) {
      *reinterpret_cast<float4*>(row + c) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else if (MODE == GN_SHIFT && c < width) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j >= 0 && c + j < width) row[c + j] = v[4 * i + j];
    }
  }
}
template <int E, int MODE>
__device__ __forceinline__ void gn_add(float (&v)[E], const float* row, int width, int G, int t, int off) {
  float o[E];
  gn_load<E, MODE>(o, row, width, G, t, off);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = o[e] + v[e];
}
// The weights of this thread's columns; ones where there is no vector.
template <int E, int MODE>
__device__ __forceinline__ void gn_weights(float (&v)[E], const float* w, int width, int G, int t, int off) {
  if (w && MODE == GN_SHIFT) {         // the vectors do not start like the rows
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = gn_column<MODE>(e, G, t, off);
      v[e] = c >= 0 && c < width ? __ldg(w + c) : 0.f;
    }
  } else if (w) {
    gn_load<E, MODE>(v, w, width, G, t, 0);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 1.f;
  }
}
// v[e] = act(v[e]) with the choice outside the loop
template <int E>
__device__ __forceinline__ void gn_act_all(int act, float (&v)[E]) {
  if (act == 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = gn_act(0, v[e]);
  } else if (act == 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = gn_act(1, v[e]);
  } else if (act == 2) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = gn_act(2, v[e]);
  } else if (act == 3) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = gn_act(3, v[e]);
  }
}
// Column sums in shared memory: vector (of 4 floats, or of E fewer) number i of thread t at i * threads + t.
template <int E>
struct GnVector {
  using type = float4;
};
template <>
struct GnVector<2> {
  using type = float2;
};
template <>
struct GnVector<1> {
  using type = float;
};
template <int E>
__device__ __forceinline__ void gn_sum_into(typename GnVector<E>::type* s, const float (&v)[E]) {
  if constexpr (E == 1) {
    *s += v[0];
  } else if constexpr (E == 2) {
    float2 q = *s;
    q.x += v[0]; q.y += v[1];
    *s = q;
  } else {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      float4 q = s[i * blockDim.x];
      q.x += v[4 * i]; q.y += v[4 * i + 1]; q.z += v[4 * i + 2]; q.w += v[4 * i + 3];
      s[i * blockDim.x] = q;
    }
  }
}

// A row on its way into L2: its 128-byte lines are asked for by the row's threads.  Not with 4 floats a thread, where the
// instructions of a row count.
__device__ __forceinline__ void gn_prefetch(const float* row, int width, int G, int t) {
  for (int c = 32 * t; c < width; c += 32 * G) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + c));
}

// Sum over the G threads of a row, in a fixed order; valid in all of them.  All threads of the block
// call it together.
__device__ __forceinline__ float gn_row_sum(float v, int G, float* smem) {
  v = warp_sum(v);
  if (G == 32) return v;
  const int warp = threadIdx.x >> 5, wpr = G >> 5;      // warps per row
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[warp] = v;
  __syncthreads();
  const int first = warp - warp % wpr;
  float s = 0.f;
  for (int w = 0; w < wpr; ++w) s += smem[first + w];
  return s;
}

template <int E, int MODE, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS > 256 ? 1 : E == 16 ? 3 : 4) gated_norm_forward_kernel(GatedNorm p, int G) {
  // the weights in registers from the start: where their loads are single, or few rows leave their latency bare
  constexpr bool KEEP = MODE == GN_SHIFT || E <= 4;
  __shared__ float red[32];
  const int t = threadIdx.x & (G - 1), per_block = blockDim.x / G;
  const float inv_width = 1.f / (float)p.width;
  const int64_t row_first = (int64_t)blockIdx.x * per_block + threadIdx.x / G;
  const int off = MODE == GN_SHIFT ? (int)((reinterpret_cast<uintptr_t>(p.x + row_first * p.ld_x) >> 2) & 3) : 0;
  float w_post[KEEP ? E : 1], w_scale[KEEP ? E : 1], w_pre[KEEP ? E : 1];
  if constexpr (KEEP) {
    gn_weights<E, MODE>(w_post, p.w_post, p.width, G, t, off);
    gn_weights<E, MODE>(w_scale, p.scale, p.width, G, t, off);
    gn_weights<E, MODE>(w_pre, p.w_pre, p.width, G, t, off);
  }
  auto weights = [&](float (&v)[E], const float* from, const float* kept) {
    if constexpr (KEEP) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = kept[e];
    } else {
      gn_weights<E, MODE>(v, from, p.width, G, t, off);
    }
  };
  for (int64_t row0 = (int64_t)blockIdx.x * per_block; row0 < p.rows; row0 += (int64_t)gridDim.x * per_block) {
    const int64_t row = row0 + threadIdx.x / G;
    const bool live = row < p.rows;
    float x[E], y[E], g[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = y[e] = g[e] = 0.f;
    if (live) {
      gn_load<E, MODE>(x, p.x + row * p.ld_x, p.width, G, t, off);
      if (p.y) {
        gn_load<E, MODE>(y, p.y + row * p.ld_y, p.width, G, t, off);
        if (p.gate) gn_load<E, MODE>(g, p.gate + row * p.ld_gate, p.width, G, t, off);
      }
      const int64_t next = row + (int64_t)gridDim.x * per_block;
      if (E > 4 && next < p.rows) {
        gn_prefetch(p.x + next * p.ld_x, p.width, G, t);
        if (p.y) gn_prefetch(p.y + next * p.ld_y, p.width, G, t);
        if (p.gate) gn_prefetch(p.gate + next * p.ld_gate, p.width, G, t);
      }
    }
    if (p.y) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += y[e] * y[e];
      const float r = gn_rsqrt(gn_row_sum(s, G, red) * inv_width + p.eps);
      if (p.gate) {
        gn_act_all<E>(p.act, g);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = y[e] * r * g[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] *= r;
      }
      weights(g, p.w_post, w_post);
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] *= g[e];
      weights(g, p.scale, w_scale);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] += y[e] * g[e];
      if (live) {
        gn_store<E, MODE>(x, p.x_out + row * p.ld_x_out, p.width, G, t, off);
        if (t == 0 && p.r_post) p.r_post[row] = r;
      }
    }
    if (p.h_out) {
      weights(g, p.w_pre, w_pre);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += x[e] * x[e];
      const float r = gn_rsqrt(gn_row_sum(s, G, red) * inv_width + p.eps);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = x[e] * r * g[e];
      if (live) {
        gn_store<E, MODE>(x, p.h_out + row * p.ld_h_out, p.width, G, t, off);
        if (t == 0 && p.r_pre) p.r_pre[row] = r;
      }
    }
  }
}

// Shared memory: three vectors of column sums for each group of G threads (gn_sum_into).
template <int E, int MODE, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS > 256 ? 1 : E == 16 ? 2 : 3) gated_norm_backward_kernel(GatedNormGrad p, int G) {
  constexpr bool KEEP = MODE == GN_SHIFT || E <= 4;
  using Sum = typename GnVector<E>::type;
  constexpr int W = E < 4 ? E : 4, N = E / W;      // floats of a vector, vectors of a thread
  extern __shared__ float4 sum_space[];
  Sum* sums = reinterpret_cast<Sum*>(sum_space);
  __shared__ float red[32];
  const int t = threadIdx.x & (G - 1), per_block = blockDim.x / G;
  Sum* s_post = sums + threadIdx.x;
  Sum* s_scale = s_post + N * blockDim.x;
  Sum* s_pre = s_scale + N * blockDim.x;
#pragma unroll
  for (int i = 0; i < N; ++i) s_post[i * blockDim.x] = s_scale[i * blockDim.x] = s_pre[i * blockDim.x] = Sum();
  const float inv_width = 1.f / (float)p.width;
  const int64_t row_first = (int64_t)blockIdx.x * per_block + threadIdx.x / G;
  const int off = MODE == GN_SHIFT ? (int)((reinterpret_cast<uintptr_t>(p.dx + row_first * p.ld_dx) >> 2) & 3) : 0;
  float w_post[KEEP ? E : 1], w_scale[KEEP ? E : 1], w_pre[KEEP ? E : 1];
  if constexpr (KEEP) {
    gn_weights<E, MODE>(w_post, p.w_post, p.width, G, t, off);
    gn_weights<E, MODE>(w_scale, p.scale, p.width, G, t, off);
    gn_weights<E, MODE>(w_pre, p.w_pre, p.width, G, t, off);
  }
  auto weights = [&](float (&v)[E], const float* from, const float* kept) {
    if constexpr (KEEP) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = kept[e];
    } else {
      gn_weights<E, MODE>(v, from, p.width, G, t, off);
    }
  };
  for (int64_t row0 = (int64_t)blockIdx.x * per_block; row0 < p.rows; row0 += (int64_t)gridDim.x * per_block) {
    const int64_t row = row0 + threadIdx.x / G;
    const bool live = row < p.rows;
    float x[E], y[E], g[E], d[E], h[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = y[e] = g[e] = d[e] = h[e] = 0.f;
    float r_pre = 0.f, r_post = 0.f;
    if (live) {
      if (p.dh) {
        gn_load<E, MODE>(h, p.dh + row * p.ld_dh, p.width, G, t, off);
        gn_load<E, MODE>(x, p.x_out + row * p.ld_x_out, p.width, G, t, off);
        r_pre = p.r_pre[row];
      }
      if (p.dx_out) gn_load<E, MODE>(d, p.dx_out + row * p.ld_dx_out, p.width, G, t, off);
      if (p.y) {
        gn_load<E, MODE>(y, p.y + row * p.ld_y, p.width, G, t, off);
        if (p.gate) gn_load<E, MODE>(g, p.gate + row * p.ld_gate, p.width, G, t, off);
        r_post = p.r_post[row];
      }
      const int64_t next = row + (int64_t)gridDim.x * per_block;
      if (E > 4 && next < p.rows) {
        if (p.dh) {
          gn_prefetch(p.dh + next * p.ld_dh, p.width, G, t);
          gn_prefetch(p.x_out + next * p.ld_x_out, p.width, G, t);
        }
        if (p.dx_out) gn_prefetch(p.dx_out + next * p.ld_dx_out, p.width, G, t);
        if (p.y) gn_prefetch(p.y + next * p.ld_y, p.width, G, t);
        if (p.gate) gn_prefetch(p.gate + next * p.ld_gate, p.width, G, t);
      }
    }
    if (p.dh) {
      float s = 0.f, w[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[e] *= r_pre;
        w[e] = h[e] * x[e];
      }
      gn_sum_into<E>(s_pre, w);
      weights(w, p.w_pre, w_pre);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[e] *= w[e];
        s += h[e] * x[e];
      }
      const float m = gn_row_sum(s, G, red) * inv_width;
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] += r_pre * (h[e] - x[e] * m);
    }
    if (live) {
      if (p.accumulate && p.dx != p.dx_out) {      // in the place of dx_out, what is there is in d already
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = d[e];
        gn_add<E, MODE>(o, p.dx + row * p.ld_dx, p.width, G, t, off);
        gn_store<E, MODE>(o, p.dx + row * p.ld_dx, p.width, G, t, off);
      } else {
        gn_store<E, MODE>(d, p.dx + row * p.ld_dx, p.width, G, t, off);
      }
    }
    if (p.y) {
      // x and h are free: x = act(gate), h = n = y^ w_post, w the weights
      float s = 0.f, w[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = p.gate ? g[e] : 1.f;
      if (p.gate) gn_act_all<E>(p.act, x);
      weights(w, p.w_post, w_post);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        y[e] *= r_post;
        h[e] = y[e] * w[e];
        g[e] = d[e] * x[e] * h[e];
      }
      gn_sum_into<E>(s_scale, g);
      weights(g, p.scale, w_scale);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        d[e] *= g[e];                                             // G scale
        g[e] = d[e] * h[e];                                       // without act'
        d[e] *= x[e];
        h[e] = d[e] * y[e];
        d[e] *= w[e];
        s += d[e] * y[e];
      }
      if (p.gate) {
        if (p.act == 0) {
#pragma unroll
          for (int e = 0; e < E; ++e) g[e] *= gn_act_deriv(0, x[e]);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) g[e] *= gn_act_deriv(p.act, x[e]);
        }
      }
      gn_sum_into<E>(s_post, h);
      const float m = gn_row_sum(s, G, red) * inv_width;
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = r_post * (d[e] - y[e] * m);
      if (live) {
        if (p.accumulate) gn_add<E, MODE>(d, p.dy + row * p.ld_dy, p.width, G, t, off);
        gn_store<E, MODE>(d, p.dy + row * p.ld_dy, p.width, G, t, off);
        if (p.gate) {
          if (p.accumulate) gn_add<E, MODE>(g, p.dgate + row * p.ld_dgate, p.width, G, t, off);
          gn_store<E, MODE>(g, p.dgate + row * p.ld_dgate, p.width, G, t, off);
        }
      }
    }
  }
  if (!p.partials) return;
  if (MODE == GN_SHIFT) {       // each group's columns are its own: a row of partial sums for each
    if (row_first >= p.rows) return;
    float* out = p.partials + row_first * 3 * p.width;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = gn_column<MODE>(e, G, t, off);
      if (c < 0 || c >= p.width) continue;
      out[c] = reinterpret_cast<const float*>(s_post + e / W * blockDim.x)[e % W];
      out[p.width + c] = reinterpret_cast<const float*>(s_scale + e / W * blockDim.x)[e % W];
      out[2 * p.width + c] = reinterpret_cast<const float*>(s_pre + e / W * blockDim.x)[e % W];
    }
    return;
  }
  __syncthreads();
  if (threadIdx.x < G) {      // the groups of the block, in order
    float* out = p.partials + (int64_t)blockIdx.x * 3 * p.width;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = gn_column<MODE>(e, G, t, 0);
      if (c >= p.width) continue;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const float* col = reinterpret_cast<const float*>(sums + (int64_t)(k * N + e / W) * blockDim.x + t) + e % W;
        float s = 0.f;
        for (int q = 0; q < per_block; ++q) s += col[W * q * G];
        out[(int64_t)k * p.width + c] = s;
      }
    }
  }
}

// out[c] (+)= sum over the partial rows of column c, for the three vectors laid side by side.  32
// columns x 16 slices of rows per block; the slices are added in order.
__global__ void __launch_bounds__(512) gated_norm_sums_kernel(const float* partials, int rows, int width, float* dw_post, float* dscale,
                                                              float* dw_pre, int accumulate) {
  __shared__ float part[16][33];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const int64_t cols = 3 * (int64_t)width;
  float s = 0.f;
  if (c < cols)
#pragma unroll 8
    for (int b = slice; b < rows; b += 16) s += partials[(int64_t)b * cols + c];
  part[slice][lane] = s;
  __syncthreads();
  if (slice || c >= cols) return;
  s = part[0][lane];
#pragma unroll
  for (int k = 1; k < 16; ++k) s += part[k][lane];
  const int which = (int)(c / width);
  float* out = which == 0 ? dw_post : which == 1 ? dscale : dw_pre;
  if (!out) return;
  out += c - (int64_t)which * width;
  *out = accumulate ? *out + s : s;
}

// How a call goes: the mode, threads per row (G) and floats per thread (E), the fewest threads (a warp at least) that
// hold the row in 16 floats each, or 8 where registers are short (single loads with their bounds, kept weights); blocks.
struct GnShape {
  int mode, G, E, threads, per_block, blocks;
};
static GnShape gn_geometry(int64_t rows, int width, int mode, bool backward) {
  GnShape s;
  s.mode = mode;
  const int span = width + (mode == GN_SHIFT ? 3 : 0);
  s.E = mode == GN_SINGLE && span <= 64 ? (span <= 32 ? 1 : 2) : span <= 128 ? 4 : (span <= 256 || (mode != GN_VEC && span <= 8192)) ? 8 : 16;
  // Few rows: a call is the latency of one row, which is shorter with 4 floats a thread, as long as all rows are resident
  // at once (128 x 1000: forward 4.6 -> 3.3 us, backward 14.9 -> 7.0; 592 x 1000: 4.8 -> 4.5, 15.5 -> 12.7; forward of 400 x 2000
  // 5.6 -> 8.2, of 64 x 4096 4.6 -> 5.5: fewer, wider blocks fit).
  if (mode != GN_SINGLE && span <= (mode == GN_VEC && backward ? 4096 : 2048)) {
    int G = 32;
    while (G * 4 < span) G *= 2;
    if (ceil_div(rows, std::max(1, 256 / G)) * (backward ? 1 : std::max(1, G / 256)) <= 4 * state().sm_count) s.E = 4;
  }
  s.G = 32;
  while (s.G * s.E < span) s.G *= 2;
  s.threads = std::max(s.G, 256);
  s.per_block = s.threads / s.G;
  const int per_sm = s.threads > 256 ? 1 : backward ? (s.E == 16 ? 2 : 3) : (s.E == 16 ? 3 : 4);      // as the launch bounds
  s.blocks = (int)std::min<int64_t>(ceil_div(rows, s.per_block), (int64_t)state().sm_count * per_sm);
  // a thread's rows are blocks * per_block apart: in the shifted form a multiple of 4
  if (mode == GN_SHIFT && s.blocks * (int64_t)s.per_block < rows)
    while (s.blocks * s.per_block % 4) --s.blocks;
  return s;
}
// Widths of the shifted form: not those that four single loads a lane hold (295099 x 83: forward 198 us shifted, 155 single,
// backward 329 and 243: the ends of the rows cost more instructions than there are loads); a row and its offset fit 512 or
// 1024 threads with 8 floats each, and fill most of them (2000 x 5001: forward 124 -> 91 us, backward 198 -> 129 against single
// loads; 500 x 4095: 19 -> 29, 36 -> 44).
static bool gn_shiftable(int width) { return width > 128 && (width + 3 <= 4096 || (width >= 4800 && width + 3 <= 8192)); }
// Rows of partial sums that a backward call leaves.
static int64_t gn_partial_rows(int64_t rows, const GnShape& s) {
  return s.mode == GN_SHIFT ? std::min<int64_t>(rows, (int64_t)s.blocks * s.per_block) : s.blocks;
}
// arrays: row-pitched operands of the call (NULL left out), vectors: the weights
static GnShape gn_shape(int64_t rows, int width, std::initializer_list<std::pair<const void*, int64_t>> arrays,
                        std::initializer_list<const void*> vectors, bool backward) {
  bool vec = width % 4 == 0, alike = true;
  uintptr_t start = 4;
  int64_t pitch = 0;
  for (const auto& a : arrays) {
    if (!a.first) continue;
    const uintptr_t at = ((uintptr_t)a.first >> 2) & 3;
    vec = vec && at == 0 && a.second % 4 == 0;
    alike = alike && (start == 4 || (at == start && (a.second - pitch) % 4 == 0));
    start = at;
    pitch = a.second;
  }
  for (const void* v : vectors) vec = vec && aligned16(v);
  // up to 64 columns a float or two a lane, whatever the alignment (1000000 x 32: forward 358 -> 297 us, backward 566 -> 438;
  // x 30: 445 -> 294, 690 -> 435; 254292 x 42: 125 -> 96, 194 -> 149, against four)
  return gn_geometry(rows, width, width <= 64 ? GN_SINGLE : vec ? GN_VEC : alike && gn_shiftable(width) ? GN_SHIFT : GN_SINGLE, backward);
}

}  // namespace b200

using namespace b200;

// Rows of up to 4096 values (2045 in the shifted form): blocks of 256 threads; wider ones: one row for a block of 512 or 1024.
// Few rows of 2049 to 4096 values take `FEW` (4 floats a thread in the backward pass only).
#define GN_KERNELS(KERNEL, FEW)                                                                                          \
  (s.mode == GN_VEC ? (s.threads == 1024 ? (s.E == 4 ? FEW : KERNEL<16, GN_VEC, 1024>)                                   \
                       : s.threads == 512 ? (s.E == 4 ? KERNEL<4, GN_VEC, 512> : KERNEL<16, GN_VEC, 512>)                \
                       : s.E == 4 ? KERNEL<4, GN_VEC, 256> : s.E == 8 ? KERNEL<8, GN_VEC, 256> : KERNEL<16, GN_VEC, 256>) \
   : s.mode == GN_SHIFT ? (s.threads == 1024 ? KERNEL<8, GN_SHIFT, 1024>                                                 \
                           : s.threads == 512 ? (s.E == 4 ? KERNEL<4, GN_SHIFT, 512> : KERNEL<8, GN_SHIFT, 512>)         \
                           : s.E == 4 ? KERNEL<4, GN_SHIFT, 256> : KERNEL<8, GN_SHIFT, 256>)                             \
   : s.threads == 1024 ? (s.E == 8 ? KERNEL<8, GN_SINGLE, 1024> : KERNEL<16, GN_SINGLE, 1024>)                           \
   : s.threads == 512 ? KERNEL<8, GN_SINGLE, 512>                                                                        \
                      : s.E == 1 ? KERNEL<1, GN_SINGLE, 256> : s.E == 2 ? KERNEL<2, GN_SINGLE, 256>                      \
                      : s.E == 4 ? KERNEL<4, GN_SINGLE, 256> : KERNEL<8, GN_SINGLE, 256>)

B200_API int b200_gated_norm_forward(const b200_gated_norm_args* args) {
  if (int rc = require_ready()) return rc;
  B200_REQUIRE(args, "gated norm: NULL arguments");
  const auto& [x, y, gate, w_post, scale, w_pre, x_out, h_out, r_post, r_pre, rows, width, ld_x, ld_y, ld_gate, ld_x_out, ld_h_out, eps, act] = *args;
  B200_REQUIRE(rows >= 0 && width >= 0, "negative extent");
  B200_REQUIRE(width <= GN_MAX_WIDTH, "gated norm: rows of more than %d values are not supported", GN_MAX_WIDTH);
  B200_REQUIRE(act >= 0 && act <= 4, "unknown activation %d", act);
  B200_REQUIRE(eps >= 0.f, "gated norm: epsilon must not be negative");
  if (rows == 0 || width == 0) return B200_OK;
  B200_REQUIRE(x && (y || h_out), "gated norm: nothing to compute");
  B200_REQUIRE(!y || x_out, "gated norm: a block output needs x_out");
  B200_REQUIRE(y || !gate, "gated norm: a gate needs a block output");
  B200_REQUIRE(ld_x >= width && (!y || (ld_y >= width && ld_x_out >= width)) && (!gate || ld_gate >= width) && (!h_out || ld_h_out >= width),
               "gated norm: leading dimension too small");
  B200_REQUIRE(rows == 1 || ((x_out != x || !y || ld_x_out == ld_x) && (h_out != y || !y || ld_h_out == ld_y)),
               "gated norm: in place, both arrays have the same row pitch");
  GatedNorm p = {x, y, gate, w_post, scale, w_pre, x_out, h_out, r_post, r_pre, rows, ld_x, ld_y, ld_gate, ld_x_out, ld_h_out,
                 (int)width, act, eps};
  const GnShape s = gn_shape(rows, (int)width, {{x, ld_x}, {y, ld_y}, {gate, ld_gate}, {y ? x_out : nullptr, ld_x_out}, {h_out, ld_h_out}},
                             {w_post, scale, w_pre}, false);
  (GN_KERNELS(gated_norm_forward_kernel, (gated_norm_forward_kernel<16, GN_VEC, 1024>)))<<<s.blocks, s.threads, 0, state().stream>>>(p, s.G);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

B200_API int64_t b200_gated_norm_scratch_floats(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0 || width > GN_MAX_WIDTH) return 0;
  int64_t most = 0;       // the form depends on the pointers
  for (int mode : {GN_SINGLE, GN_VEC, GN_SHIFT})
    if (mode != GN_SHIFT || gn_shiftable(width)) most = std::max(most, gn_partial_rows(rows, gn_geometry(rows, (int)width, mode, true)));
  return most * 3 * width;
}

B200_API int b200_gated_norm_backward(const float* x_out, const float* y, const float* gate, const float* w_post, const float* scale,
                                      const float* w_pre, const float* r_post, const float* r_pre, const float* dx_out, const float* dh,
                                      float* dx, float* dy, float* dgate, float* dw_post, float* dscale, float* dw_pre, int64_t rows,
                                      int64_t width, int64_t ld_x_out, int64_t ld_y, int64_t ld_gate, int64_t ld_dx_out, int64_t ld_dh,
                                      int64_t ld_dx, int64_t ld_dy, int64_t ld_dgate, int act, int accumulate, float* scratch,
                                      int64_t scratch_floats) {
  if (int rc = require_ready()) return rc;
  B200_REQUIRE(rows >= 0 && width >= 0, "negative extent");
  B200_REQUIRE(width <= GN_MAX_WIDTH, "gated norm: rows of more than %d values are not supported", GN_MAX_WIDTH);
  B200_REQUIRE(act >= 0 && act <= 4, "unknown activation %d", act);
  const bool sums = dw_post || dscale || dw_pre;
  if (width == 0) return B200_OK;
  if (rows == 0) {   // empty sums
    if (!accumulate)
      for (float* v : {dw_post, dscale, dw_pre})
        if (v) B200_CUDA(cudaMemsetAsync(v, 0, (size_t)width * sizeof(float), state().stream));
    return B200_OK;
  }
  B200_REQUIRE(dx && (y || dh), "gated norm: nothing to compute");
  B200_REQUIRE(!dh || (x_out && r_pre), "gated norm: dh needs x_out and r_pre");
  B200_REQUIRE(!y || (r_post && dy), "gated norm: a block output needs r_post and dy");
  B200_REQUIRE(!gate || (y && dgate), "gated norm: a gate needs a block output and dgate");
  B200_REQUIRE(ld_dx >= width && (!dh || (ld_dh >= width && ld_x_out >= width)) && (!dx_out || ld_dx_out >= width) &&
                   (!y || (ld_y >= width && ld_dy >= width)) && (!gate || (ld_gate >= width && ld_dgate >= width)),
               "gated norm: leading dimension too small");
  B200_REQUIRE(rows == 1 || dx != dx_out || ld_dx == ld_dx_out, "gated norm: in place, both arrays have the same row pitch");
  B200_REQUIRE(!sums || (scratch && scratch_floats >= b200_gated_norm_scratch_floats(rows, width)), "gated norm: scratch too small");
  GatedNormGrad p = {x_out, y, gate, w_post, scale, w_pre, r_post, r_pre, dx_out, dh, dx, dy, dgate, sums ? scratch : nullptr, rows,
                     ld_x_out, ld_y, ld_gate, ld_dx_out, ld_dh, ld_dx, ld_dy, ld_dgate, (int)width, act, accumulate ? 1 : 0};
  const GnShape s = gn_shape(rows, (int)width,
                             {{dh ? x_out : nullptr, ld_x_out}, {y, ld_y}, {gate, ld_gate}, {dx_out, ld_dx_out}, {dh, ld_dh}, {dx, ld_dx},
                              {y ? dy : nullptr, ld_dy}, {gate ? dgate : nullptr, ld_dgate}},
                             {w_post, scale, w_pre}, true);
  const size_t smem = (size_t)3 * s.E * s.threads * sizeof(float);
  auto kernel = GN_KERNELS(gated_norm_backward_kernel, (gated_norm_backward_kernel<4, GN_VEC, 1024>));
  // 48 KiB and more of dynamic shared memory has to be asked for (the static part counts too)
  if (smem >= 48 * 1024) B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<s.blocks, s.threads, smem, state().stream>>>(p, s.G);
  B200_LAUNCH_CHECK();
  if (sums) {
    const int partial_rows = (int)gn_partial_rows(rows, s);
    gated_norm_sums_kernel<<<(unsigned)ceil_div(3 * width, 32), 512, 0, state().stream>>>(scratch, partial_rows, (int)width, dw_post, dscale, dw_pre,
                                                                                          accumulate ? 1 : 0);
    B200_LAUNCH_CHECK();
  }
  return B200_OK;
}
