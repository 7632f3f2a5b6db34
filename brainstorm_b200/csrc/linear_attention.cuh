// Decayed linear attention: what its kernels share.
//
// For each sequence b and head h, with the head's decay l:
//
//   S_t = l S_{t-1} + k_t (x) v_t        o_t = scale * q_t S_t          t = 0 .. n_b - 1
//
// Forward and all three gradients are ONE operator with other roles and directions, a `LaRun`:
//
//   out:  Q = q,  K = k, V = v,   first token first, S starts from state       (o_scale = scale)
//   dq:   Q = do, K = v, V = k,   first token first, S starts from state^T     (o_scale = scale)
//   dk:   Q = v,  K = do, V = q,  last token first,  S starts from dstate_out^T  (k_scale = scale)
//   dv:   Q = k,  K = q, V = do,  last token first,  S starts from dstate_out   (k_scale = scale), ends as dstate
//
// because S_t and its gradient M_t = sum_{s >= t} l^{s-t} scale q_s (x) do_s + l^{n-1-t} dstate_out obey the
// same recurrence in opposite directions.  Going backwards the incoming state counts undecayed at the
// first token visited, and the outgoing one is decayed once more (state enters S_0 with a factor l).
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int LA_MAX_DIM = 128;

struct LaStrides {      // of a (T, B, heads, d) array with contiguous d; `div`: heads of the operator per head of the array
  int64_t t, b, h;
  int div;
};
struct LaRun {
  const float *q, *k, *v;
  float* o;
  LaStrides qs, ks, vs, os;
  const float* s_in;     // (B, H, dk, dv), or (B, H, dv, dk) with s_in_t; NULL = zeros
  float* s_out;          // (B, H, dk, dv) or NULL
  int s_in_t, reverse, accumulate;
  int dk, dv;
  float k_scale, o_scale;
};
struct LaCommon {
  const float *decay, *lengths;   // (H), (B) or NULL = all T
  int T, B, H;
};

// Tokens of sequence b: its length truncated like a label and held to [0, T]; a NaN counts as 0.
__device__ __forceinline__ int la_length(const LaCommon& c, int b) {
  if (!c.lengths) return c.T;
  const float f = c.lengths[b];
  return !(f >= 1.f) ? 0 : f >= (float)c.T ? c.T : (int)f;
}

// l^e, e >= 0, by squarings in 64 bits
__device__ __forceinline__ double la_power(double l, int e) {
  double f = 1.;
  for (; e > 0; e >>= 1, l *= l)
    if (e & 1) f *= l;
  return f;
}

// x, or the largest number in the place of an infinity: a factor beyond the range of float32 may meet zeros (tokens without
// a key, a state that is zero still), which an infinity would turn into NaN.
__device__ __forceinline__ float la_finite(float x) { return fabsf(x) > 3.402823466e38f ? copysignf(3.402823466e38f, x) : x; }
__device__ __forceinline__ float la_power32(double l, int e) { return la_finite((float)la_power(l, e)); }

int la_recurrent(const LaCommon& c, const LaRun* runs, int count);                      // linear_attention.cu
int la_chunked(const LaCommon& c, const LaRun* runs, int count, float* work);           // linear_attention_chunks.cu
int64_t la_chunked_work(int64_t T, int64_t BH, int dk, int dv, bool backward);          // floats
}  // namespace b200
