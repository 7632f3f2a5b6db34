// Decayed linear attention, chunked form: for prompts and training.
//
// A chunk of up to C = 64 tokens, i, j inside it, S the state before it:
//
//   o_i = sum_{j <= i} l^{i-j} (q_i . k_j) v_j + l^{i+1} q_i S        S' = l^n S + sum_j l^{n-1-j} k_j (x) v_j
//
// One block of four warps walks the chunks of one (sequence, head), or of a segment of them, for up to 64
// columns of v, with the state in registers.  All four products run on mma.sync.m16n8k16 in fp32 accuracy:
// every operand x is scaled by a power of two (per tile, per row for q and the scores) and split into two
// half-precision parts, hi = fp16(x), lo = fp16(x - hi), 22 bits together, and a product is hi.hi + hi.lo +
// lo.hi.  A value more than 2^17 below the largest of its tile begins to lose bits (the error stays below
// 2^-39 of that largest value).
//
// Why mma.sync and not tcgen05: a chunk's products are 64 x 64 x d with a mask, weights and a new split
// between them; the split and the weights want the accumulators in the registers that compute them, where
// mma.sync leaves them, and the masked half of the scores is skipped in steps of 16.  Measured here:
// mma.sync fp16 555 TFLOP/s (185 of fp32 accuracy), tf32 277 (92 in three products).  With d = 64 a token
// and head needs 13.3 k products, 40 clocks of an SM, against 44 clocks of HBM time for its 1 KiB.
//
// Few sequences and heads: the time axis is cut into segments.  A first pass computes what each segment adds
// to the state, a second one hands the state through, then all segments run side by side.
//
// Bound: HBM and the tensor pipe about evenly at d = 64, the tensor pipe at d = 128.
#include <cuda_fp16.h>

#include <algorithm>

#include "linear_attention.cuh"

namespace b200 {

constexpr int LC = 64;                // tokens in a chunk
constexpr int LC_COLS = 64;           // columns of v in a block
constexpr int LC_THREADS = 128;

struct LaChunkRun {
  LaRun r;
  float* work;                        // segment states [segment][b * H + h][dk][dv], or NULL when there is one segment
  int work_t, state_pass;             // the run whose layout `work` has is the transposed one; run takes part in the state pass
};
struct LaChunkRuns {
  LaChunkRun run[3];
};

__device__ __forceinline__ uint32_t lc_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void lc_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lc_ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lc_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// c += (ah + al)(bh + bl) without al.bl; the small terms first
__device__ __forceinline__ void lc_mma3(float (&c)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], uint32_t bh0, uint32_t bh1, uint32_t bl0,
                                        uint32_t bl1) {
  lc_mma(c, al, bh0, bh1);
  lc_mma(c, ah, bl0, bl1);
  lc_mma(c, ah, bh0, bh1);
}
__device__ __forceinline__ uint32_t lc_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// two values as (hi, hi) and (lo, lo)
__device__ __forceinline__ void lc_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = lc_bits(h);
  lo = lc_bits(__floats2half2_rn(x - f.x, y - f.y));
}
// |x|, 0 for a value that is not finite (which must not decide a scale)
__device__ __forceinline__ float lc_size(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// The power of two that takes a largest value m into [2^13, 2^14); *inv its reciprocal.
__device__ __forceinline__ float lc_scale(float m, float* inv) {
  const int e = (int)(__float_as_uint(m) >> 23) - 127;
  const int k = min(13 - e, 126);         // 2^126 and its reciprocal are both normal numbers
  *inv = __uint_as_float((uint32_t)(127 - k) << 23);
  return __uint_as_float((uint32_t)(127 + k) << 23);
}
// Byte offset of 16-byte group `g` of row `row` in a tile of halves with `pitch` bytes a row: groups are
// permuted within their 128 bytes by the row, so that eight rows of one column meet eight bank groups.
__device__ __forceinline__ uint32_t lc_at(int row, int g, int pitch) { return (uint32_t)(row * pitch + ((g ^ (row & 7)) << 4)); }

// Rows of d values from a (T, B, heads, d) array: row `i` of the tile is token `tok(i)`; zero outside.
template <bool VEC>
__device__ __forceinline__ float4 lc_row4(const float* row, int c, int d) {
  if (VEC) return c < d ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(c < d ? row[c] : 0.f, c + 1 < d ? row[c + 1] : 0.f, c + 2 < d ? row[c + 2] : 0.f, c + 3 < d ? row[c + 3] : 0.f);
}
__device__ __forceinline__ float lc_max4(float m, float4 x) {
  return fmaxf(m, fmaxf(fmaxf(lc_size(x.x), lc_size(x.y)), fmaxf(lc_size(x.z), lc_size(x.w))));
}
__device__ __forceinline__ void lc_put4(uint8_t* hi, uint8_t* lo, int row, int c, int pitch, float4 x, float s) {
  uint32_t h0, l0, h1, l1;
  lc_split(x.x * s, x.y * s, h0, l0);
  lc_split(x.z * s, x.w * s, h1, l1);
  const uint32_t at = lc_at(row, c >> 3, pitch) + ((c & 4) << 1);
  *reinterpret_cast<uint2*>(hi + at) = make_uint2(h0, h1);
  *reinterpret_cast<uint2*>(lo + at) = make_uint2(l0, l1);
}

template <int DK>
struct LcSmem {
  static constexpr int KP = DK * 2, VP = LC_COLS * 2;      // row pitch in bytes
  static constexpr int Q_HI = 0, Q_LO = LC * KP, K_HI = 2 * LC * KP, K_LO = 3 * LC * KP, V_HI = 4 * LC * KP, V_LO = V_HI + LC * VP,
                       S_HI = V_LO + LC * VP, S_LO = S_HI + DK * VP, BYTES = S_LO + DK * VP;
};

// DK: 64 or 128, the largest dk the block can hold.  VEC: 128-bit global loads.  STATE_ONLY: the state pass.
template <int DK, bool VEC, bool STATE_ONLY>
__global__ void __launch_bounds__(LC_THREADS, DK == 64 ? 3 : 2) la_chunk_kernel(LaCommon c, LaChunkRuns runs, int segments, int seg_tokens, int max_slabs) {
  using L = LcSmem<DK>;
  constexpr int MT = DK / 64;                        // 16-row tiles of the state in a warp
  constexpr int LPR = DK / 4, RPP = LC_THREADS / LPR;   // lanes per row of k, rows in a pass
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ float pw[LC + 1];                       // powers of the decay
  __shared__ float q_inv[LC];                        // 1 / scale of each row of q
  __shared__ float red[3][4];

  const LaChunkRun& cr = runs.run[blockIdx.y];
  const LaRun& p = cr.r;
  int id = blockIdx.x;
  const int slab = id % max_slabs;
  id /= max_slabs;
  const int seg = id % segments, bh = id / segments;
  const int slabs = (p.dv + LC_COLS - 1) / LC_COLS;
  if (slab >= slabs || (STATE_ONLY && !cr.state_pass)) return;
  const int b = bh / c.H, h = bh % c.H;
  const int n_all = la_length(c, b);
  const int64_t first = (int64_t)seg * seg_tokens;                 // steps of this segment
  const int64_t limit = min((int64_t)c.T, first + seg_tokens);
  const int64_t n_end = min((int64_t)n_all, limit);
  // the slab's columns: a multiple of 8, all slabs about equally wide
  const int width = ((p.dv + slabs - 1) / slabs + 7) & ~7;
  const int v0 = slab * width, dv = min(width, p.dv - v0), dk = p.dk;
  const int nt_n = (dv + 7) >> 3;                                  // 8-column tiles in use
  const int ks_n = (dk + 15) >> 4;                                 // 16-deep steps over dk
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t2 = (lane & 3) * 2;
  const float l = c.decay[h];
  const int64_t states = (int64_t)dk * p.dv;

  const float* q = STATE_ONLY ? nullptr : p.q + (int64_t)b * p.qs.b + (int64_t)(h / p.qs.div) * p.qs.h;
  const float* k = p.k + (int64_t)b * p.ks.b + (int64_t)(h / p.ks.div) * p.ks.h;
  const float* v = p.v + (int64_t)b * p.vs.b + (int64_t)(h / p.vs.div) * p.vs.h + v0;
  float* o = STATE_ONLY ? nullptr : p.o + (int64_t)b * p.os.b + (int64_t)(h / p.os.div) * p.os.h + v0;

  if (tid <= LC) pw[tid] = tid == 0 ? 1.f : (float)pow((double)l, (double)tid);

  // state: 16-row tiles w and w + 4 (rows 16 (w + 4 m) + g and + 8), columns 8 nt + t2, t2 + 1
  float S[MT][8][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[m][nt][e] = 0.f;
  auto row_of = [&](int m, int e) { return 16 * (w + 4 * m) + g + (e >> 1) * 8; };
  auto col_of = [&](int nt, int e) { return 8 * nt + t2 + (e & 1); };
  if (!STATE_ONLY) {
    const float* s0 = segments > 1 ? cr.work + ((int64_t)seg * c.B * c.H + bh) * states : p.s_in ? p.s_in + bh * states : nullptr;
    const int tr = segments > 1 ? cr.work_t : p.s_in_t;
    if (s0)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = row_of(m, e), j = col_of(nt, e);
            if (i < dk && j < dv) S[m][nt][e] = tr ? s0[(int64_t)(v0 + j) * dk + i] : s0[(int64_t)i * p.dv + v0 + j];
          }
  }
  bool undecayed = !STATE_ONLY && p.reverse && seg == 0;          // the incoming state counts in full at the first token

  for (int64_t c0 = first; c0 < n_end; c0 += LC) {
    const int n = (int)min((int64_t)LC, n_end - c0);
    auto token = [&](int i) { return p.reverse ? n_all - 1 - (c0 + i) : c0 + i; };
    // ---- load k and v, the scales of k, v and the state
    float4 kr[LC / RPP], vr[8];
    float mk = 0.f, mv = 0.f, ms = 0.f;
    const int kc = (tid % LPR) * 4, vc = (tid & 15) * 4;
#pragma unroll
    for (int it = 0; it < LC / RPP; ++it) {
      const int i = it * RPP + tid / LPR;
      kr[it] = i < n ? lc_row4<VEC>(k + token(i) * p.ks.t, kc, dk) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int i = it * 8 + (tid >> 4);
      vr[it] = i < n ? lc_row4<VEC>(v + token(i) * p.vs.t, vc, dv) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int it = 0; it < LC / RPP; ++it) mk = lc_max4(mk, kr[it]);
#pragma unroll
    for (int it = 0; it < 8; ++it) mv = lc_max4(mv, vr[it]);
    if (!STATE_ONLY)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) ms = fmaxf(ms, lc_size(S[m][nt][e]));
    mk = warp_max(mk);
    mv = warp_max(mv);
    if (!STATE_ONLY) ms = warp_max(ms);
    if (lane == 0) {
      red[0][w] = mk;
      red[1][w] = mv;
      red[2][w] = ms;
    }
    __syncthreads();      // scales in place; every warp is done with the tiles of the chunk before
    float k_inv, v_inv, s_inv, w_inv = 1.f;
    const float k_s = lc_scale(fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])), &k_inv);
    const float v_s = lc_scale(fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3])), &v_inv);
    const float s_s = lc_scale(fmaxf(fmaxf(red[2][0], red[2][1]), fmaxf(red[2][2], red[2][3])), &s_inv);
    // weights above one (a decay above one) are taken back below two
    float w_s = 1.f;
    const float w_max = fabsf(pw[n - 1]);
    if (w_max > 1.f) {
      w_s = lc_scale(w_max, &w_inv) * 0x1p-13f;
      w_inv *= 0x1p13f;
    }
#pragma unroll
    for (int it = 0; it < LC / RPP; ++it) lc_put4(sm + L::K_HI, sm + L::K_LO, it * RPP + tid / LPR, kc, L::KP, kr[it], k_s);
#pragma unroll
    for (int it = 0; it < 8; ++it) {
      const int i = it * 8 + (tid >> 4);
      float f = v_s;
      if (STATE_ONLY) f = i < n ? v_s * (pw[n - 1 - i] * w_s) : 0.f;
      if (STATE_ONLY) lc_put4(sm + L::Q_HI, sm + L::Q_LO, i, vc, L::KP, vr[it], f);
      else lc_put4(sm + L::V_HI, sm + L::V_LO, i, vc, L::VP, vr[it], f);
    }
    float acc_o[8][4];
    if (!STATE_ONLY) {
      // ---- q, scaled by row
#pragma unroll 8
      for (int it = 0; it < LC / RPP; ++it) {
        const int i = it * RPP + tid / LPR;
        const float4 x = i < n ? lc_row4<VEC>(q + token(i) * p.qs.t, kc, dk) : make_float4(0.f, 0.f, 0.f, 0.f);
        float m = lc_max4(0.f, x), inv;
#pragma unroll
        for (int s = 1; s < LPR; s <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        const float sc = lc_scale(m, &inv);
        lc_put4(sm + L::Q_HI, sm + L::Q_LO, i, kc, L::KP, x, sc);
        if (tid % LPR == 0) q_inv[i] = inv;
      }
      // ---- the state
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            uint32_t hi, lo;
            lc_split(S[m][nt][e] * s_s, S[m][nt][e + 1] * s_s, hi, lo);
            const uint32_t at = lc_at(row_of(m, e), nt, L::VP) + t2 * 2;
            *reinterpret_cast<uint32_t*>(sm + L::S_HI + at) = hi;
            *reinterpret_cast<uint32_t*>(sm + L::S_LO + at) = lo;
          }
    }
    __syncthreads();      // all tiles in place
    if (!STATE_ONLY) {
      const int i0 = 16 * w;                          // this warp's tokens
      if (i0 < n) {
        // ---- scores of the tokens up to this warp's, and q S, in one walk over dk
        float P[8][4];
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) P[nt][e] = acc_o[nt][e] = 0.f;
#pragma unroll 2
        for (int ks = 0; ks < ks_n; ++ks) {
          uint32_t qh[4], ql[4];
          const uint32_t qa = lc_at(i0 + (lane & 15), 2 * ks + (lane >> 4), L::KP);
          lc_ldmatrix(qh, lc_smem(sm + L::Q_HI) + qa);
          lc_ldmatrix(ql, lc_smem(sm + L::Q_LO) + qa);
#pragma unroll
          for (int jt = 0; jt < 4; ++jt)
            if (jt <= w) {
              uint32_t bh_[4], bl_[4];
              const uint32_t ka = lc_at(16 * jt + (lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1), L::KP);
              lc_ldmatrix(bh_, lc_smem(sm + L::K_HI) + ka);
              lc_ldmatrix(bl_, lc_smem(sm + L::K_LO) + ka);
              lc_mma3(P[2 * jt], qh, ql, bh_[0], bh_[1], bl_[0], bl_[1]);
              lc_mma3(P[2 * jt + 1], qh, ql, bh_[2], bh_[3], bl_[2], bl_[3]);
            }
#pragma unroll
          for (int vt = 0; vt < 4; ++vt)
            if (2 * vt < nt_n) {
              uint32_t bh_[4], bl_[4];
              const uint32_t sa = lc_at(16 * ks + (lane & 15), 2 * vt + (lane >> 4), L::VP);
              lc_ldmatrix_t(bh_, lc_smem(sm + L::S_HI) + sa);
              lc_ldmatrix_t(bl_, lc_smem(sm + L::S_LO) + sa);
              lc_mma3(acc_o[2 * vt], qh, ql, bh_[0], bh_[1], bl_[0], bl_[1]);
              lc_mma3(acc_o[2 * vt + 1], qh, ql, bh_[2], bh_[3], bl_[2], bl_[3]);
            }
        }
        // ---- weights and mask, then the scores' own scale for each row
        float m0 = 0.f, m1 = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
          if (nt < 2 * w + 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int apart = i0 + g + (e >> 1) * 8 - col_of(nt, e);
              P[nt][e] = apart >= 0 ? P[nt][e] * pw[apart < 0 ? 0 : apart] : 0.f;
            }
            m0 = fmaxf(m0, fmaxf(lc_size(P[nt][0]), lc_size(P[nt][1])));
            m1 = fmaxf(m1, fmaxf(lc_size(P[nt][2]), lc_size(P[nt][3])));
          }
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, s));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, s));
        }
        float p_inv0, p_inv1;
        const float p_s0 = lc_scale(m0, &p_inv0), p_s1 = lc_scale(m1, &p_inv1);
        // ---- scores times v
        float acc_p[8][4];
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc_p[nt][e] = 0.f;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
          if (jt <= w) {
            uint32_t ah[4], al[4];
            lc_split(P[2 * jt][0] * p_s0, P[2 * jt][1] * p_s0, ah[0], al[0]);
            lc_split(P[2 * jt][2] * p_s1, P[2 * jt][3] * p_s1, ah[1], al[1]);
            lc_split(P[2 * jt + 1][0] * p_s0, P[2 * jt + 1][1] * p_s0, ah[2], al[2]);
            lc_split(P[2 * jt + 1][2] * p_s1, P[2 * jt + 1][3] * p_s1, ah[3], al[3]);
#pragma unroll
            for (int vt = 0; vt < 4; ++vt)
              if (2 * vt < nt_n) {
                uint32_t bh_[4], bl_[4];
                const uint32_t va = lc_at(16 * jt + (lane & 15), 2 * vt + (lane >> 4), L::VP);
                lc_ldmatrix_t(bh_, lc_smem(sm + L::V_HI) + va);
                lc_ldmatrix_t(bl_, lc_smem(sm + L::V_LO) + va);
                lc_mma3(acc_p[2 * vt], ah, al, bh_[0], bh_[1], bl_[0], bl_[1]);
                lc_mma3(acc_p[2 * vt + 1], ah, al, bh_[2], bh_[3], bl_[2], bl_[3]);
              }
          }
        // ---- out
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = i0 + g + 8 * half;
          if (i < n) {
            const float qi = q_inv[i];
            const float f_s = p.o_scale * pw[i + (undecayed ? 0 : 1)];
            const float f_p = p.o_scale * p.k_scale;
            const float p_inv = half ? p_inv1 : p_inv0;
            float* row = o + token(i) * p.os.t;
#pragma unroll
            for (int nt = 0; nt < 8; ++nt)
              if (nt < nt_n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int j = 8 * nt + t2 + e;
                  const float x = acc_o[nt][2 * half + e] * s_inv * qi * f_s + acc_p[nt][2 * half + e] * p_inv * v_inv * (qi * k_inv) * f_p;
                  if (j < dv) row[j] = p.accumulate ? row[j] + x : x;
                }
          }
        }
      }
      // ---- v times its weights, over this warp's rows of q (which only this warp has read)
      __syncwarp();
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int i = 16 * w + 2 * it + (lane >> 4), cc = (lane & 15) * 4;
        const uint32_t at = lc_at(i, cc >> 3, L::VP) + ((cc & 4) << 1);
        const uint2 hi = *reinterpret_cast<const uint2*>(sm + L::V_HI + at), lo = *reinterpret_cast<const uint2*>(sm + L::V_LO + at);
        const float f = i < n ? pw[n - 1 - i] * w_s : 0.f;
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi.x)), a2 = __half22float2(*reinterpret_cast<const __half2*>(&lo.x));
        const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&hi.y)), d2 = __half22float2(*reinterpret_cast<const __half2*>(&lo.y));
        lc_put4(sm + L::Q_HI, sm + L::Q_LO, i, cc, L::KP, make_float4(a.x + a2.x, a.y + a2.y, d.x + d2.x, d.y + d2.y), f);
      }
      __syncthreads();    // weighted v in place; the state's tile has been read
    }
    // ---- the state after the chunk
    const float keep = pw[n - (undecayed ? 1 : 0)];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r0 = 16 * (w + 4 * m);
      if (r0 < dk) {
        float acc[8][4];
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
          if (16 * kt < n) {
            uint32_t ah[4], al[4];
            const uint32_t ka = lc_at(16 * kt + (lane & 7) + ((lane >> 4) << 3), (r0 >> 3) + ((lane >> 3) & 1), L::KP);
            lc_ldmatrix_t(ah, lc_smem(sm + L::K_HI) + ka);
            lc_ldmatrix_t(al, lc_smem(sm + L::K_LO) + ka);
#pragma unroll
            for (int vt = 0; vt < 4; ++vt)
              if (2 * vt < nt_n) {
                uint32_t bh_[4], bl_[4];
                const uint32_t va = lc_at(16 * kt + (lane & 15), 2 * vt + (lane >> 4), L::KP);
                lc_ldmatrix_t(bh_, lc_smem(sm + L::Q_HI) + va);
                lc_ldmatrix_t(bl_, lc_smem(sm + L::Q_LO) + va);
                lc_mma3(acc[2 * vt], ah, al, bh_[0], bh_[1], bl_[0], bl_[1]);
                lc_mma3(acc[2 * vt + 1], ah, al, bh_[2], bh_[3], bl_[2], bl_[3]);
              }
          }
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[m][nt][e] = keep * S[m][nt][e] + acc[nt][e] * (k_inv * w_inv) * v_inv * p.k_scale;
      }
    }
    undecayed = false;
  }

  if (!STATE_ONLY && !p.accumulate)       // tokens behind the end of the sequence
    for (int64_t t = max((int64_t)n_all, first); t < limit; ++t)
      for (int j = tid; j < dv; j += LC_THREADS) o[t * p.os.t + j] = 0.f;
  float* out = STATE_ONLY ? cr.work + ((int64_t)seg * c.B * c.H + bh) * states : segments == 1 && p.s_out ? p.s_out + bh * states : nullptr;
  if (out) {
    const float f = (!STATE_ONLY && p.reverse && n_all > 0) ? l : 1.f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = row_of(m, e), j = col_of(nt, e);
          if (i < dk && j < dv) out[(int64_t)i * p.dv + v0 + j] = f * S[m][nt][e];
        }
  }
}

// The state through the segments: work[seg] (what segment seg adds) becomes the state before it.
__global__ void __launch_bounds__(256) la_segments_kernel(LaCommon c, LaChunkRuns runs, int segments, int seg_tokens) {
  const LaChunkRun& cr = runs.run[blockIdx.z];
  if (!cr.state_pass) return;
  const LaRun& p = cr.r;
  const int bh = blockIdx.y, b = bh / c.H, h = bh % c.H;
  const int64_t states = (int64_t)p.dk * p.dv, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= states) return;
  const int n = la_length(c, b);
  const double l = c.decay[h];
  float S = 0.f;
  if (p.s_in) S = p.s_in[bh * states + (p.s_in_t ? (e % p.dv) * p.dk + e / p.dv : e)];
  const float full = (float)pow(l, (double)seg_tokens);
  for (int s = 0; s < segments; ++s) {
    float* at = cr.work + ((int64_t)s * c.B * c.H + bh) * states + e;
    const float add = *at;
    *at = S;
    const int64_t left = (int64_t)n - (int64_t)s * seg_tokens;
    const int count = (int)(left < 0 ? 0 : left < seg_tokens ? left : seg_tokens);
    const int times = (p.reverse && s == 0 && count > 0) ? count - 1 : count;
    const float f = times == 0 ? 1.f : times == seg_tokens ? full : (float)pow(l, (double)times);
    if (count > 0) S = f * S + add;
  }
  if (p.s_out) p.s_out[bh * states + e] = (p.reverse && n > 0) ? (float)l * S : S;
}

// Segments for `blocks` blocks of one segment: as many as use the resident blocks of the GPU best, where
// every pass over a part costs its chunks and a state pass costs about half of that.
static int lc_segments(int64_t T, int64_t blocks, int resident) {
  const int64_t chunks = ceil_div(T, LC);
  int best = 1;
  double best_cost = (double)chunks * (double)ceil_div(blocks, resident);
  for (int s = 2; s <= 64 && 2 * s <= chunks; ++s) {
    const int64_t per = ceil_div(chunks, s);
    const double cost = 1.5 * (double)per * (double)ceil_div(blocks * s, resident) + 2.0;
    if (cost < 0.9 * best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}
static int lc_dk(const LaRun* runs, int count) {
  int dk = 0;
  for (int i = 0; i < count; ++i) dk = std::max(dk, runs[i].dk);
  return dk <= 64 ? 64 : 128;
}
struct LcPlan {
  int segments, seg_tokens, slabs, dk;
};
static LcPlan lc_plan(int64_t T, int64_t BH, int dk, int dv_max, int count) {
  LcPlan p;
  p.dk = dk <= 64 ? 64 : 128;
  p.slabs = (int)ceil_div(dv_max, LC_COLS);
  p.segments = lc_segments(T, BH * p.slabs * count, state().sm_count * (p.dk == 64 ? 3 : 2));
  p.seg_tokens = (int)(ceil_div(ceil_div(T, LC), p.segments) * LC);
  p.segments = (int)ceil_div(T, p.seg_tokens);
  return p;
}
// Work for the chunked form: the segment states of the runs that have a state pass.
int64_t la_chunked_work(int64_t T, int64_t BH, int dk, int dv, bool backward) {
  const LcPlan p = backward ? lc_plan(T, BH, std::max(dk, dv), std::max(dk, dv), 3) : lc_plan(T, BH, dk, dv, 1);
  return p.segments > 1 ? (int64_t)(backward ? 2 : 1) * p.segments * BH * dk * dv : 0;
}

template <int DK>
static int lc_launch(const LaCommon& c, const LaChunkRuns& all, int count, const LcPlan& p, bool vec) {
  const cudaStream_t st = state().stream;
  const size_t smem = LcSmem<DK>::BYTES;
  const int64_t blocks = (int64_t)c.B * c.H * p.segments * p.slabs;
  B200_REQUIRE(blocks < (1ll << 31), "linear attention: extent too large");
  auto main_kernel = vec ? la_chunk_kernel<DK, true, false> : la_chunk_kernel<DK, false, false>;
  B200_CUDA(cudaFuncSetAttribute(main_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if (p.segments > 1) {
    auto state_kernel = vec ? la_chunk_kernel<DK, true, true> : la_chunk_kernel<DK, false, true>;
    B200_CUDA(cudaFuncSetAttribute(state_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    state_kernel<<<dim3((unsigned)blocks, (unsigned)count), LC_THREADS, smem, st>>>(c, all, p.segments, p.seg_tokens, p.slabs);
    B200_LAUNCH_CHECK();
    const int64_t most = (int64_t)all.run[0].r.dk * all.run[0].r.dv;      // the same product for every run
    la_segments_kernel<<<dim3((unsigned)ceil_div(most, 256), (unsigned)((int64_t)c.B * c.H), (unsigned)count), 256, 0, st>>>(c, all, p.segments, p.seg_tokens);
    B200_LAUNCH_CHECK();
  }
  main_kernel<<<dim3((unsigned)blocks, (unsigned)count), LC_THREADS, smem, st>>>(c, all, p.segments, p.seg_tokens, p.slabs);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

// Forward: one run.  Backward: dq, dk, dv in that order; dk's state is dv's transposed.
int la_chunked(const LaCommon& c, const LaRun* runs, int count, float* work) {
  const bool backward = count == 3;
  const int64_t BH = (int64_t)c.B * c.H, states = (int64_t)runs[0].dk * runs[0].dv;
  int dv_max = 0;
  bool vec = true;
  for (int i = 0; i < count; ++i) {
    dv_max = std::max(dv_max, runs[i].dv);
    for (const float* a : {runs[i].q, runs[i].k, runs[i].v}) vec = vec && aligned16(a);
    for (const LaStrides* s : {&runs[i].qs, &runs[i].ks, &runs[i].vs}) vec = vec && s->t % 4 == 0 && s->b % 4 == 0 && s->h % 4 == 0;
    // a slab starts at a multiple of 8 columns: aligned when the rows are
    vec = vec && runs[i].dk % 4 == 0 && runs[i].dv % 4 == 0;
  }
  const LcPlan p = lc_plan(c.T, BH, lc_dk(runs, count), dv_max, count);
  B200_REQUIRE(BH <= 65535 || p.segments == 1, "linear attention: extent too large");
  LaChunkRuns all = {};
  for (int i = 0; i < count; ++i) all.run[i] = LaChunkRun{runs[i], p.segments > 1 ? work : nullptr, 0, 1};
  if (backward && p.segments > 1) {
    all.run[2].work = work + p.segments * BH * states;
    all.run[1].work = all.run[2].work;
    all.run[1].work_t = 1;
    all.run[1].state_pass = 0;
  }
  return p.dk == 64 ? lc_launch<64>(c, all, count, p, vec) : lc_launch<128>(c, all, count, p, vec);
}

}  // namespace b200
