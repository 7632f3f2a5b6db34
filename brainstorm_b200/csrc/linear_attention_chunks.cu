// Decayed linear attention, chunked form: for prompts and training.
//
// A chunk of up to C = 64 tokens, i, j inside it, S the state before it:
//
//   o_i = sum_{j <= i} l^{i-j} (q_i . k_j) v_j + l^{i+1} q_i S        S' = l^n S + sum_j l^{n-1-j} k_j (x) v_j
//
// One block of four warps walks the chunks of one (sequence, head), or of a segment of them, for up to 64
// columns of v, with the state in registers.  All four products run on mma.sync.m16n8k16 in fp32 accuracy:
// every operand x is scaled by a power of two and split into two half-precision parts, hi = fp16(x), lo = fp16(x - hi), 22
// bits together, and a product is hi.hi + hi.lo + lo.hi.  A scale belongs to one token's row of q, k or v, to one row of
// scores, or to the state: what a token's output does not depend on, a later token above all, does not decide a scale
// that it is computed with.  The scales of k and v are taken back where the scores get their decay, and enter the weights
// with which a chunk's keys and values are added to the state.  A value more than 2^17 below the largest of its row, or of
// the state, begins to lose bits (the error stays below 2^-38 of that largest value).
//
// Why mma.sync and not tcgen05: a chunk's products are 64 x 64 x d with a mask, weights and a new split
// between them; the split and the weights want the accumulators in the registers that compute them, where
// mma.sync leaves them, and the masked half of the scores is skipped in steps of 16.  Measured here:
// mma.sync fp16 555 TFLOP/s (185 of fp32 accuracy), tf32 277 (92 in three products).  With d = 64 a token
// and head needs 13.3 k products, 40 clocks of an SM, against 44 clocks of HBM time for its 1 KiB.  A form of
// the outputs on tcgen05 (128 tokens a block, q and the scores in tensor memory, the states of all chunks from the
// state pass) was right and slower: 8192 x 2 x 16 heads of 128 913 us against 626, since a block that fills
// shared memory loads, splits, multiplies and stores in a row, and every chunk's state goes through HBM.
//
// Few sequences and heads: the time axis is cut into segments.  A first pass computes what each segment adds
// to the state, a second one hands the state through, then all segments run side by side.
//
// Bound: neither memory nor the tensor pipe (33 and 26 % of the clocks at d = 128 and 64) but the latency between
// dependent instructions: registers and shared memory let two or three blocks onto an SM, two or three warps a
// scheduler, which issue in 38 to 46 % of the clocks.  Measured: 8192 x 2 x 16 heads of 128 626 us (state pass 165, handing
// through 20, outputs 435), HBM time 83; 100 x 128 x 16 heads of 64 with gradients 511 us, HBM time 114; 1999 x 6 x 12 heads
// of 48 and 80 over 4, ragged, with gradients 596 to 628 us, HBM time 39.  (With one scale for all of a chunk's keys, and one for
// its values, 598, 454 and 570 us, but a token then lost bits to later ones.)
//
// Errors against 64 bits, of |out| and of the gradients together: 4 to 7e-7, two to three times those of sums in float32:
// sums on the tensor core truncate.
#include <cuda_fp16.h>

#include <algorithm>

#include "half_split.cuh"
#include "linear_attention.cuh"

namespace b200 {

constexpr int LC = 64;                // tokens in a chunk
constexpr int LC_COLS = 64;           // columns of v in a block
constexpr int LS_THREADS = 256;       // of the state pass

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
// Not volatile: a function of registers, which the compiler may move between the loads.
__device__ __forceinline__ void lc_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four 8-column tiles: c += (ah + al)(bh + bl) without al.bl, the small terms first.  Term by term, so that four
// products lie between two that add to the same registers.
__device__ __forceinline__ void lc_mma3(float (&c0)[4], float (&c1)[4], float (&c2)[4], float (&c3)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4],
                                        const uint32_t (&bh)[8], const uint32_t (&bl)[8]) {
  lc_mma(c0, al, bh[0], bh[1]);
  lc_mma(c1, al, bh[2], bh[3]);
  lc_mma(c2, al, bh[4], bh[5]);
  lc_mma(c3, al, bh[6], bh[7]);
  lc_mma(c0, ah, bl[0], bl[1]);
  lc_mma(c1, ah, bl[2], bl[3]);
  lc_mma(c2, ah, bl[4], bl[5]);
  lc_mma(c3, ah, bl[6], bl[7]);
  lc_mma(c0, ah, bh[0], bh[1]);
  lc_mma(c1, ah, bh[2], bh[3]);
  lc_mma(c2, ah, bh[4], bh[5]);
  lc_mma(c3, ah, bh[6], bh[7]);
}
// the same for two tiles
__device__ __forceinline__ void lc_mma3(float (&c0)[4], float (&c1)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const uint32_t (&bh)[8],
                                        const uint32_t (&bl)[8]) {
  lc_mma(c0, al, bh[0], bh[1]);
  lc_mma(c1, al, bh[2], bh[3]);
  lc_mma(c0, ah, bl[0], bl[1]);
  lc_mma(c1, ah, bl[2], bl[3]);
  lc_mma(c0, ah, bh[0], bh[1]);
  lc_mma(c1, ah, bh[2], bh[3]);
}
// c (16 x 8 N) += a (16 x 16) b, b the 16 rows from `row` and the 8-column tiles from nt0 of a tile of 64 columns; those
// from nt_n on do not count
template <int N>
__device__ __forceinline__ void lc_rows(float (&c)[N][4], const uint32_t (&ah)[4], const uint32_t (&al)[4], uint32_t hi, uint32_t lo, int row, int lane,
                                        int nt0, int nt_n) {
#pragma unroll
  for (int nt = 0; nt < N; nt += 4)
    if (nt0 + nt < nt_n) {
      uint32_t bh[8], bl[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t at = (uint32_t)((row + (lane & 15)) * 128 + (((nt0 + nt + 2 * u + (lane >> 4)) ^ (lane & 7)) << 4));
        lc_ldmatrix_t(*reinterpret_cast<uint32_t(*)[4]>(bh + 4 * u), hi + at);
        lc_ldmatrix_t(*reinterpret_cast<uint32_t(*)[4]>(bl + 4 * u), lo + at);
      }
      lc_mma3(c[nt], c[nt + 1], c[nt + 2], c[nt + 3], ah, al, bh, bl);
    }
}
__device__ __forceinline__ uint32_t lc_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// (hi + lo) of two values
__device__ __forceinline__ float2 lc_join(uint32_t hi, uint32_t lo) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi)), b = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2(a.x + b.x, a.y + b.y);
}
// |x|, 0 for a value that is not finite (which must not decide a scale)
__device__ __forceinline__ float lc_size(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// 2^k, k from -126 to 127
__device__ __forceinline__ float lc_pow2(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }
// The power of two that takes a largest value m into [2^13, 2^14); *inv its reciprocal.
__device__ __forceinline__ float lc_scale(float m, float* inv) {
  const int e = (int)(__float_as_uint(m) >> 23) - 127;
  const int k = min(13 - e, 126);         // 2^126 and its reciprocal are both normal numbers
  *inv = lc_pow2(-k);
  return lc_pow2(k);
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
// Largest magnitude; FINITE leaves out what is not finite (a NaN is never taken).
template <bool FINITE>
__device__ __forceinline__ float lc_max4(float m, float4 x) {
  if (FINITE) return fmaxf(m, fmaxf(fmaxf(lc_size(x.x), lc_size(x.y)), fmaxf(lc_size(x.z), lc_size(x.w))));
  return fmaxf(fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
}
template <bool FINITE, int N>
__device__ __forceinline__ float lc_max(const float4 (&x)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = lc_max4<FINITE>(m, x[i]);
  return m;
}
template <bool FINITE, int M, int N>
__device__ __forceinline__ float lc_max(const float (&x)[M][N][4]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) m = lc_max4<FINITE>(m, make_float4(x[i][j][0], x[i][j][1], x[i][j][2], x[i][j][3]));
  return m;
}
#define LC_INF __int_as_float(0x7f800000)
// The scales of the rows of a tile, two rows in a word: biased exponents of the powers of two that take a row's largest finite
// magnitude into (2^13, 2^14], 2^126 at most; 254 for a row of zeros.  A row lies in LANES neighbouring lanes, one
// float4 each; all rows' shuffles together.  All lanes of the warp call it.
template <int LANES, int N>
__device__ __forceinline__ void lc_row_scales(uint32_t (&e)[N / 2], const float4 (&x)[N]) {
  float m[N];
  bool inf = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    m[i] = lc_max4<false>(0.f, x[i]);
    inf = inf || m[i] == LC_INF;
  }
  if (__any_sync(0xffffffffu, inf)) {      // an infinity must not decide a scale
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = lc_max4<true>(0.f, x[i]);
  }
  // exponents rounded up, from 1 on for all but zero
#pragma unroll
  for (int i = 0; i < N / 2; ++i) e[i] = __byte_perm(__float_as_uint(m[2 * i]) + 0x7fffffu >> 7, __float_as_uint(m[2 * i + 1]) + 0x7fffffu >> 7, 0x7632) & 0x01ff01ffu;
#pragma unroll
  for (int s = 1; s < LANES; s <<= 1)
#pragma unroll
    for (int i = 0; i < N / 2; ++i) e[i] = __vmaxu2(e[i], __shfl_xor_sync(0xffffffffu, e[i], s));
#pragma unroll
  for (int i = 0; i < N / 2; ++i) e[i] = __vminu2(0x010c010cu - e[i], 0x00fd00fdu) + __vseteq2(e[i], 0);      // 268 - e is 141 - (e - 127) biased
}
template <int N>
__device__ __forceinline__ uint32_t lc_row(const uint32_t (&e)[N], int i) { return i & 1 ? e[i / 2] >> 16 : e[i / 2] & 0xffff; }
__device__ __forceinline__ float lc_biased(uint32_t b) { return __uint_as_float(b << 23); }
// 1 / scale, 0 for a row of zeros
__device__ __forceinline__ float lc_inverse(uint32_t b) { return lc_biased(254 - b); }
// The weights of a chunk's n tokens in the state after it, l^(n-1-j) k_inv[j] v_inv[j], as u0 (token `lane`), u1 (token 32 + `lane`),
// all below 2, times 2^(*f0's and *f1's exponents): taken together a weight may be outside the range of float32, and the
// largest decides the scale, so that a token that the decay has removed does not count, nor one without a key or a value.
__device__ __forceinline__ void lc_weights(float& u0, float& u1, float& f0, float& f1, const float* pw, const float* k_inv, const float* v_inv, int n, int lane) {
  auto exponent = [](float x) { return (int)(__float_as_uint(x) >> 23 & 255) - 127; };
  const float k0 = k_inv[lane], k1 = k_inv[lane + 32], v0 = v_inv[lane], v1 = v_inv[lane + 32];
  const float p0 = lane < n && k0 != 0.f && v0 != 0.f ? pw[n - 1 - lane] : 0.f, p1 = lane + 32 < n && k1 != 0.f && v1 != 0.f ? pw[n - 33 - lane] : 0.f;
  const int e0 = exponent(k0) + exponent(v0), e1 = exponent(k1) + exponent(v1);
  const int top = __reduce_max_sync(0xffffffffu, max(p0 != 0.f ? e0 + exponent(p0) : -1000, p1 != 0.f ? e1 + exponent(p1) : -1000));
  // in two factors: where a power of the decay is far below one, the other exponents may be far above the largest sum
  auto scaled = [](float p, int e) {
    const int half = e >> 1;
    return p * lc_pow2(max(-126, min(127, half))) * lc_pow2(max(-126, min(127, e - half)));
  };
  u0 = scaled(p0, e0 - top);
  u1 = scaled(p1, e1 - top);
  f0 = lc_pow2(max(-126, min(127, top >> 1)));
  f1 = lc_pow2(max(-126, min(127, top - (top >> 1))));
}
__device__ __forceinline__ void lc_put4(uint8_t* hi, uint8_t* lo, int row, int c, int pitch, float4 x, float s) {
  uint32_t h0, l0, h1, l1;
  split_halves(x.x * s, x.y * s, h0, l0);
  split_halves(x.z * s, x.w * s, h1, l1);
  const uint32_t at = lc_at(row, c >> 3, pitch) + ((c & 4) << 1);
  *reinterpret_cast<uint2*>(hi + at) = make_uint2(h0, h1);
  *reinterpret_cast<uint2*>(lo + at) = make_uint2(l0, l1);
}

template <int DK>
struct LcSmem {
  static constexpr int KP = DK * 2, VP = LC_COLS * 2;      // row pitch in bytes; hi and lo parts of q, k, v and the state
  static constexpr int Q_HI = 0, Q_LO = LC * KP, K_HI = 2 * LC * KP, K_LO = 3 * LC * KP, V_HI = 4 * LC * KP, V_LO = V_HI + LC * VP,
                       S_HI = V_LO + LC * VP, S_LO = S_HI + DK * VP, BYTES = S_LO + DK * VP;
};

// A warp computes the outputs of 16 tokens of a chunk and keeps a quarter of the state in its registers; all four load and
// split the tiles.  With THREADS = 256 two warps have the same tokens and rows of the state and half of the columns each; both
// compute the scores.  DK: 64 or 128, the largest dk the block can hold.  VEC: 128-bit global loads.
template <int DK, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 1 : DK == 64 ? 3 : 2) la_chunk_kernel(LaCommon c, LaChunkRuns runs, int segments, int seg_tokens, int max_slabs, int sms) {
  using L = LcSmem<DK>;
  constexpr int MT = DK / 64;                        // 16-row tiles of the state in a warp
  constexpr int NT = 8 * 128 / THREADS;           // 8-column tiles of a warp
  constexpr int LPR = DK / 4, RPP = THREADS / LPR;   // lanes per row of k, rows in a pass
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ float pw_pad[16 + LC + 1];              // powers of the decay, zeros before
  __shared__ __align__(8) float k_inv[LC], v_inv[LC];      // 1 / scale of each row
  __shared__ uint8_t q_scale[LC];                    // biased exponents of the scales of q (a float each would not leave room for two blocks)
  __shared__ float red[THREADS / 32];
  const float* pw = pw_pad + 16;

  const LaChunkRun& cr = runs.run[blockIdx.y];
  const LaRun& p = cr.r;
  int id = blockIdx.x;
  const int slab = id % max_slabs;
  id /= max_slabs;
  const int seg = id % segments, bh = id / segments;
  const int slabs = (p.dv + LC_COLS - 1) / LC_COLS;
  if (slab >= slabs) return;
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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, w = warp & 3, nt0 = NT * (warp >> 2), g = lane >> 2, t2 = (lane & 3) * 2;
  const float l = c.decay[h];
  const int64_t states = (int64_t)dk * p.dv;

  // step s of the walk is token s, or n_all - 1 - s: a start and a signed pitch
  const int64_t tok0 = p.reverse ? n_all - 1 : 0;
  const int64_t q_t = p.reverse ? -p.qs.t : p.qs.t, k_t = p.reverse ? -p.ks.t : p.ks.t, v_t = p.reverse ? -p.vs.t : p.vs.t,
                o_t = p.reverse ? -p.os.t : p.os.t;
  const float* q = p.q + (int64_t)b * p.qs.b + (int64_t)(h / p.qs.div) * p.qs.h + tok0 * p.qs.t;
  const float* k = p.k + (int64_t)b * p.ks.b + (int64_t)(h / p.ks.div) * p.ks.h + tok0 * p.ks.t;
  const float* v = p.v + (int64_t)b * p.vs.b + (int64_t)(h / p.vs.div) * p.vs.h + v0 + tok0 * p.vs.t;
  float* o_base = p.o + (int64_t)b * p.os.b + (int64_t)(h / p.os.div) * p.os.h + v0;

  if (tid < 16 + LC + 1) pw_pad[tid] = tid < 16 ? 0.f : la_power32(l, tid - 16);
  // Later tokens meet more keys: the blocks of an SM take the rows in opposite order, so that its four schedulers get
  // about the same share.
  const int r = ((NT == 8 ? blockIdx.x / sms : warp >> 2) & 1) ? 3 - w : w, i0 = 16 * r;      // this warp's tokens
  constexpr int KN = LC / RPP, VN = LC * 16 / THREADS;             // passes over k (and q) and v
  const int kc = (tid % LPR) * 4, vc = (tid & 15) * 4;
  auto prefetch = [&](const float* a, int64_t pitch, int d, int64_t c0) {      // a tile of the next chunk on its way into L2
    constexpr int PER = THREADS / LC;                // threads of a row
    const int x = (tid % PER) * 32, i = tid / PER;
    if (c0 + LC + i < n_end)
      for (int e = x; e < d; e += 32 * PER) asm volatile("prefetch.global.L2 [%0];" ::"l"(a + (c0 + LC + i) * pitch + e));
  };

  // the state: 16-row tiles w and w + 4 (rows 16 (w + 4 m) + g and + 8), columns 8 nt + t2, t2 + 1
  auto row_of = [&](int m, int e) { return 16 * (w + 4 * m) + g + (e >> 1) * 8; };
  auto col_of = [&](int nt, int e) { return 8 * (nt0 + nt) + t2 + (e & 1); };
  float S[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[m][nt][e] = 0.f;
  {
    const float* s0 = segments > 1 ? cr.work + ((int64_t)seg * c.B * c.H + bh) * states : p.s_in ? p.s_in + bh * states : nullptr;
    const bool tr = segments > 1 ? cr.work_t : p.s_in_t;
    if (s0 && tr) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = row_of(m, e), j = col_of(nt, e);
            if (i < dk && j < dv) S[m][nt][e] = s0[(int64_t)(v0 + j) * dk + i];
          }
    } else if (s0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int i = row_of(m, e), j = col_of(nt, e);
            const float* at = s0 + (int64_t)i * p.dv + v0 + j;
            if (VEC) {
              if (i < dk && j < dv) {
                const float2 x = *reinterpret_cast<const float2*>(at);
                S[m][nt][e] = x.x;
                S[m][nt][e + 1] = x.y;
              }
            } else {
              if (i < dk && j < dv) S[m][nt][e] = at[0];
              if (i < dk && j + 1 < dv) S[m][nt][e + 1] = at[1];
            }
          }
    }
  }
  bool undecayed = p.reverse && seg == 0;            // the incoming state counts in full at the first token

  for (int64_t c0 = first; c0 < n_end; c0 += LC) {
    const int n = (int)min((int64_t)LC, n_end - c0);
    float4 kr[KN], vr[VN];
    {
      const float* kp = k + (c0 + tid / LPR) * k_t;
      const float* vp = v + (c0 + (tid >> 4)) * v_t;
#pragma unroll
      for (int it = 0; it < KN; ++it, kp += RPP * k_t)
        kr[it] = it * RPP + tid / LPR < n ? lc_row4<VEC>(kp, kc, dk) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int it = 0; it < VN; ++it, vp += LC / VN * v_t)
        vr[it] = it * (LC / VN) + (tid >> 4) < n ? lc_row4<VEC>(vp, vc, dv) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // ---- with dk up to 64 the registers hold q as well; else it follows in halves
    constexpr int QN = KN <= 8 ? KN : KN / 2;
    float4 qr[QN];
    auto load_q = [&](int it0) {
      const float* qp = q + (c0 + it0 * RPP + tid / LPR) * q_t;
#pragma unroll
      for (int it = 0; it < QN; ++it, qp += RPP * q_t)
        qr[it] = (it0 + it) * RPP + tid / LPR < n ? lc_row4<VEC>(qp, kc, dk) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    auto put_q = [&](int it0) {
      uint32_t e[QN / 2];
      lc_row_scales<LPR>(e, qr);
#pragma unroll
      for (int it = 0; it < QN; ++it) {
        const int i = (it0 + it) * RPP + tid / LPR;
        lc_put4(sm + L::Q_HI, sm + L::Q_LO, i, kc, L::KP, qr[it], lc_biased(lc_row(e, it)));
        if (tid % LPR == 0) q_scale[i] = (uint8_t)lc_row(e, it);
      }
    };
    if (QN == KN) load_q(0);
    uint32_t ke[KN / 2], ve[VN / 2];
    lc_row_scales<LPR>(ke, kr);
    lc_row_scales<16>(ve, vr);
    auto publish = [&](float m) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
      if (lane == 0) red[warp] = m;
      __syncthreads();
      m = red[0];
#pragma unroll
      for (int u = 1; u < THREADS / 32; ++u) m = fmaxf(m, red[u]);
      return m;
    };
    float s_max = publish(lc_max<false>(S));           // behind it the tiles of the chunk before are free
    if (s_max == LC_INF) {
      __syncthreads();
      s_max = publish(lc_max<true>(S));
    }
    float s_inv;
    const float s_scale = lc_scale(s_max, &s_inv);
#pragma unroll
    for (int it = 0; it < KN; ++it) {
      const int i = it * RPP + tid / LPR;
      lc_put4(sm + L::K_HI, sm + L::K_LO, i, kc, L::KP, kr[it], lc_biased(lc_row(ke, it)));
      if (tid % LPR == 0) k_inv[i] = lc_inverse(lc_row(ke, it));
    }
#pragma unroll
    for (int it = 0; it < VN; ++it) {
      const int i = it * (LC / VN) + (tid >> 4);
      lc_put4(sm + L::V_HI, sm + L::V_LO, i, vc, L::VP, vr[it], lc_biased(lc_row(ve, it)));
      if ((tid & 15) == 0) v_inv[i] = lc_inverse(lc_row(ve, it));
    }
    if (QN != KN) load_q(0);
    put_q(0);
    if (QN != KN) {
      load_q(QN);
      put_q(QN);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          uint32_t hi, lo;
          split_halves(S[m][nt][e] * s_scale, S[m][nt][e + 1] * s_scale, hi, lo);
          const uint32_t at = lc_at(row_of(m, e), nt0 + nt, L::VP) + t2 * 2;
          *reinterpret_cast<uint32_t*>(sm + L::S_HI + at) = hi;
          *reinterpret_cast<uint32_t*>(sm + L::S_LO + at) = lo;
        }
    __syncthreads();      // all tiles in place
    prefetch(k, k_t, dk, c0);
    prefetch(q, q_t, dk, c0);
    prefetch(v, v_t, dv, c0);
    if (i0 < n && nt0 < nt_n) {
      // ---- scores of the tokens up to this warp's, and q S, in one walk over dk
      float P[8][4], acc_o[NT][4];
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) P[nt][e] = acc_o[nt % NT][e] = 0.f;
#pragma unroll 1
      for (int ks = 0; ks < ks_n; ++ks) {
        uint32_t qh[4], ql[4];
        const uint32_t qa = lc_at(i0 + (lane & 15), 2 * ks + (lane >> 4), L::KP);
        lc_ldmatrix(qh, lc_smem(sm + L::Q_HI) + qa);
        lc_ldmatrix(ql, lc_smem(sm + L::Q_LO) + qa);
#pragma unroll
        for (int jt = 0; jt < 4; jt += 2)
          if (jt <= r) {
            uint32_t bh_[8], bl_[8];
            const bool both = jt < r;                   // the second 16 tokens of the 32 are not masked as a whole
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (u == 1 && !both) break;
              const uint32_t ka = lc_at(16 * (jt + u) + (lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1), L::KP);
              lc_ldmatrix(*reinterpret_cast<uint32_t(*)[4]>(bh_ + 4 * u), lc_smem(sm + L::K_HI) + ka);
              lc_ldmatrix(*reinterpret_cast<uint32_t(*)[4]>(bl_ + 4 * u), lc_smem(sm + L::K_LO) + ka);
            }
            if (both) lc_mma3(P[2 * jt], P[2 * jt + 1], P[2 * jt + 2], P[2 * jt + 3], qh, ql, bh_, bl_);
            else lc_mma3(P[2 * jt], P[2 * jt + 1], qh, ql, bh_, bl_);
          }
        lc_rows(acc_o, qh, ql, lc_smem(sm + L::S_HI), lc_smem(sm + L::S_LO), 16 * ks, lane, nt0, nt_n);
      }
      // ---- weights, the scales of q, k and v taken back, and mask, then the scores' own scale for each row.  Element
      // (nt, half, e) is apart by base - 8 (nt - half) - e tokens: the weight of half 1 is the one half 0 had a tile before.
      // Those of q and k together are out of the range of float32 only where the score is; the others one after the other.
      const float* pb = pw + (i0 + g - t2);
      const float q_inv0 = lc_inverse(q_scale[i0 + g]), q_inv1 = lc_inverse(q_scale[i0 + g + 8]);
      float m0 = 0.f, m1 = 0.f, b0 = pb[8], b1 = pb[7];
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
        if (nt < 2 * r + 2) {
          const float a0 = pb[-8 * nt], a1 = pb[-8 * nt - 1];
          float2 k2 = *reinterpret_cast<const float2*>(k_inv + 8 * nt + t2);
          const float2 v2 = *reinterpret_cast<const float2*>(v_inv + 8 * nt + t2);
          if (v2.x == 0.f) k2.x = 0.f;                 // a token without a value: its score counts nothing, however large its weight
          if (v2.y == 0.f) k2.y = 0.f;
          P[nt][0] = P[nt][0] * (q_inv0 * k2.x) * a0 * v2.x;
          P[nt][1] = P[nt][1] * (q_inv0 * k2.y) * a1 * v2.y;
          P[nt][2] = P[nt][2] * (q_inv1 * k2.x) * b0 * v2.x;
          P[nt][3] = P[nt][3] * (q_inv1 * k2.y) * b1 * v2.y;
          if (nt >= 2 * r) {                            // the tiles on the diagonal
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (g + (e >> 1) * 8 < 8 * (nt - 2 * r) + t2 + (e & 1)) P[nt][e] = 0.f;
          }
          m0 = fmaxf(m0, fmaxf(fabsf(P[nt][0]), fabsf(P[nt][1])));
          m1 = fmaxf(m1, fmaxf(fabsf(P[nt][2]), fabsf(P[nt][3])));
          b0 = a0;
          b1 = a1;
        }
      if (__any_sync(0xffffffffu, fmaxf(m0, m1) == LC_INF)) {
        m0 = m1 = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt)
          if (nt < 2 * r + 2) {
            m0 = fmaxf(m0, fmaxf(lc_size(P[nt][0]), lc_size(P[nt][1])));
            m1 = fmaxf(m1, fmaxf(lc_size(P[nt][2]), lc_size(P[nt][3])));
          }
      }
#pragma unroll
      for (int s = 1; s < 4; s <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, s));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, s));
      }
      float p_inv0, p_inv1;
      const float p_s0 = lc_scale(m0, &p_inv0), p_s1 = lc_scale(m1, &p_inv1);
      // ---- scores times v
      float acc_p[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc_p[nt][e] = 0.f;
#pragma unroll
      for (int jt = 0; jt < 4; ++jt)
        if (jt <= r) {
          uint32_t ah[4], al[4];
          split_halves(P[2 * jt][0] * p_s0, P[2 * jt][1] * p_s0, ah[0], al[0]);
          split_halves(P[2 * jt][2] * p_s1, P[2 * jt][3] * p_s1, ah[1], al[1]);
          split_halves(P[2 * jt + 1][0] * p_s0, P[2 * jt + 1][1] * p_s0, ah[2], al[2]);
          split_halves(P[2 * jt + 1][2] * p_s1, P[2 * jt + 1][3] * p_s1, ah[3], al[3]);
          lc_rows(acc_p, ah, al, lc_smem(sm + L::V_HI), lc_smem(sm + L::V_LO), 16 * jt, lane, nt0, nt_n);
        }
      // ---- out
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = i0 + g + 8 * half;
        if (i < n) {
          // the factors one after the other where their product could leave the range of float32
          const float f_o0 = s_inv * (half ? q_inv1 : q_inv0), f_o1 = la_finite(p.o_scale * pw[i + (undecayed ? 0 : 1)]);
          const float f_p0 = half ? p_inv1 : p_inv0, f_p1 = p.o_scale * p.k_scale;
          float* row = o_base + (tok0 * p.os.t + (c0 + i) * o_t);
          if (VEC && !p.accumulate) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (col_of(nt, 0) < dv)
                *reinterpret_cast<float2*>(row + col_of(nt, 0)) =
                    make_float2(acc_o[nt][2 * half] * f_o0 * f_o1 + acc_p[nt][2 * half] * f_p0 * f_p1,
                                acc_o[nt][2 * half + 1] * f_o0 * f_o1 + acc_p[nt][2 * half + 1] * f_p0 * f_p1);
          } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int j = col_of(nt, e);
                const float x = acc_o[nt][2 * half + e] * f_o0 * f_o1 + acc_p[nt][2 * half + e] * f_p0 * f_p1;
                if (j < dv) row[j] = p.accumulate ? row[j] + x : x;
              }
          }
        }
      }
    }
    // ---- the state after the chunk; each element of k is met once here and takes its weight on the way
    const float keep = pw[n - (undecayed ? 1 : 0)];
    float u0, u1, f0, f1;
    lc_weights(u0, u1, f0, f1, pw, k_inv, v_inv, n, lane);
    f1 *= p.k_scale;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r0 = 16 * (w + 4 * m);
      if (r0 < dk && nt0 < nt_n) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][e] = 0.f;
#pragma unroll(DK == 64 ? 1 : 4)      // code that follows itself soon stays in the instruction cache
        for (int kt = 0; kt < 4; ++kt)
          if (16 * kt < n) {
            uint32_t ah[4], al[4];
            const uint32_t ka = lc_at(16 * kt + (lane & 7) + ((lane >> 4) << 3), (r0 >> 3) + ((lane >> 3) & 1), L::KP);
            lc_ldmatrix_t(ah, lc_smem(sm + L::K_HI) + ka);
            lc_ldmatrix_t(al, lc_smem(sm + L::K_LO) + ka);
            {
#pragma unroll
              for (int e = 0; e < 2; ++e) {             // tokens 16 kt + 8 e + t2 and the next
                const int from = (16 * kt + 8 * e + t2) & 31;
                const float w0 = __shfl_sync(0xffffffffu, kt < 2 ? u0 : u1, from), w1 = __shfl_sync(0xffffffffu, kt < 2 ? u0 : u1, from + 1);
#pragma unroll
                for (int r = 2 * e; r < 2 * e + 2; ++r) {
                  const float2 y = lc_join(ah[r], al[r]);
                  split_halves(y.x * w0, y.y * w1, ah[r], al[r]);
                }
              }
            }
            lc_rows(acc, ah, al, lc_smem(sm + L::V_HI), lc_smem(sm + L::V_LO), 16 * kt, lane, nt0, nt_n);
          }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[m][nt][e] = keep * S[m][nt][e] + acc[nt][e] * f0 * f1;
      }
    }
    undecayed = false;
  }
  if (!p.accumulate)       // tokens behind the end of the sequence
    for (int64_t t = max((int64_t)n_all, first); t < limit; ++t)
      for (int j = tid; j < dv; j += THREADS) o_base[t * p.os.t + j] = 0.f;
  float* out = segments == 1 && p.s_out ? p.s_out + bh * states : nullptr;
  if (out) {
    const float f = (p.reverse && n_all > 0) ? l : 1.f;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int i = row_of(m, e), j = col_of(nt, e);
          float* at = out + (int64_t)i * p.dv + v0 + j;
          if (VEC) {
            if (i < dk && j < dv) *reinterpret_cast<float2*>(at) = make_float2(f * S[m][nt][e], f * S[m][nt][e + 1]);
          } else {
            if (i < dk && j < dv) at[0] = f * S[m][nt][e];
            if (i < dk && j + 1 < dv) at[1] = f * S[m][nt][e + 1];
          }
        }
  }
}

// The state pass: what a segment adds to the state, into work[segment].  Warp: 16-row tiles w and w + 4 of the state, 32 of
// the 64 columns.  The next chunk's rows are already on their way into registers while the tensor pipe works.
template <int DK, bool VEC>
__global__ void __launch_bounds__(LS_THREADS, 2) la_state_kernel(LaCommon c, LaChunkRuns runs, int segments, int seg_tokens, int max_slabs) {
  constexpr int KP = DK * 2, VP = LC_COLS * 2, K_LO = LC * KP, V_HI = 2 * LC * KP, V_LO = V_HI + LC * VP;
  constexpr int MT = DK / 64, LPR = DK / 4, RPP = LS_THREADS / LPR, KN = LC / RPP, VN = LC * 16 / LS_THREADS;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ float pw[LC + 1], k_inv[LC], v_inv[LC];

  const LaChunkRun& cr = runs.run[blockIdx.y];
  const LaRun& p = cr.r;
  int id = blockIdx.x;
  const int slab = id % max_slabs;
  id /= max_slabs;
  const int seg = id % segments, bh = id / segments;
  const int slabs = (p.dv + LC_COLS - 1) / LC_COLS;
  if (slab >= slabs || !cr.state_pass) return;
  const int b = bh / c.H, h = bh % c.H;
  const int n_all = la_length(c, b);
  const int64_t first = (int64_t)seg * seg_tokens, n_end = min((int64_t)n_all, first + seg_tokens);
  const int width = ((p.dv + slabs - 1) / slabs + 7) & ~7;
  const int v0 = slab * width, dv = min(width, p.dv - v0), dk = p.dk;
  const int nt_n = (dv + 7) >> 3;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, w = warp & 3, nt0 = 4 * (warp >> 2), g = lane >> 2, t2 = (lane & 3) * 2;
  const int64_t tok0 = p.reverse ? n_all - 1 : 0;
  const int64_t k_t = p.reverse ? -p.ks.t : p.ks.t, v_t = p.reverse ? -p.vs.t : p.vs.t;
  const int kc = (tid % LPR) * 4, vc = (tid & 15) * 4;
  const float* k = p.k + (int64_t)b * p.ks.b + (int64_t)(h / p.ks.div) * p.ks.h + (tok0 * p.ks.t + (first + tid / LPR) * k_t);
  const float* v = p.v + (int64_t)b * p.vs.b + (int64_t)(h / p.vs.div) * p.vs.h + v0 + (tok0 * p.vs.t + (first + (tid >> 4)) * v_t);
  if (tid <= LC) pw[tid] = la_power32(c.decay[h], tid);

  float4 kr[KN], vr[VN];
  auto load = [&](int64_t c0) {       // rows of the chunk at c0 (a step of this segment); zero behind the end
    const float* kp = k + (c0 - first) * k_t;
    const float* vp = v + (c0 - first) * v_t;
    const int n = (int)max((int64_t)0, min((int64_t)LC, n_end - c0));
#pragma unroll
    for (int it = 0; it < KN; ++it, kp += RPP * k_t)
      kr[it] = it * RPP + tid / LPR < n ? lc_row4<VEC>(kp, kc, dk) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int it = 0; it < VN; ++it, vp += LC / VN * v_t)
      vr[it] = it * (LC / VN) + (tid >> 4) < n ? lc_row4<VEC>(vp, vc, dv) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float S[MT][4][4], acc[MT][4][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[m][nt][e] = 0.f;
  load(first);
  for (int64_t c0 = first; c0 < n_end; c0 += LC) {
    const int n = (int)min((int64_t)LC, n_end - c0);
    uint32_t ke[KN / 2], ve[VN / 2];
    lc_row_scales<LPR>(ke, kr);
    lc_row_scales<16>(ve, vr);
#pragma unroll
    for (int it = 0; it < KN; ++it)
      if (tid % LPR == 0) k_inv[it * RPP + tid / LPR] = lc_inverse(lc_row(ke, it));
#pragma unroll
    for (int it = 0; it < VN; ++it)
      if ((tid & 15) == 0) v_inv[it * (LC / VN) + (tid >> 4)] = lc_inverse(lc_row(ve, it));
    __syncthreads();      // the scales are in place, and the tiles of the chunk before are free
    float u0, u1, f0, f1;
    lc_weights(u0, u1, f0, f1, pw, k_inv, v_inv, n, lane);
#pragma unroll
    for (int it = 0; it < KN; ++it) {
      const int i = it * RPP + tid / LPR;
      const float u = __shfl_sync(0xffffffffu, it * RPP < 32 ? u0 : u1, i & 31);
      lc_put4(sm, sm + K_LO, i, kc, KP, kr[it], lc_biased(lc_row(ke, it)) * u);
    }
#pragma unroll
    for (int it = 0; it < VN; ++it) lc_put4(sm + V_HI, sm + V_LO, it * (LC / VN) + (tid >> 4), vc, VP, vr[it], lc_biased(lc_row(ve, it)));
    __syncthreads();
    if (c0 + LC < n_end) load(c0 + LC);
    const float keep = pw[n];
    f1 *= p.k_scale;
    if (nt0 < nt_n) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][nt][e] = 0.f;
#pragma unroll 1
      for (int kt = 0; kt < 4; ++kt)
        if (16 * kt < n) {
          uint32_t bh[8], bl[8];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t va = lc_at(16 * kt + (lane & 15), nt0 + 2 * u + (lane >> 4), VP);
            lc_ldmatrix_t(*reinterpret_cast<uint32_t(*)[4]>(bh + 4 * u), lc_smem(sm + V_HI) + va);
            lc_ldmatrix_t(*reinterpret_cast<uint32_t(*)[4]>(bl + 4 * u), lc_smem(sm + V_LO) + va);
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const int r0 = 16 * (w + 4 * m);
            if (r0 >= dk) continue;
            uint32_t ah[4], al[4];
            const uint32_t ka = lc_at(16 * kt + (lane & 7) + ((lane >> 4) << 3), (r0 >> 3) + ((lane >> 3) & 1), KP);
            lc_ldmatrix_t(ah, lc_smem(sm) + ka);
            lc_ldmatrix_t(al, lc_smem(sm + K_LO) + ka);
            lc_mma3(acc[m][0], acc[m][1], acc[m][2], acc[m][3], ah, al, bh, bl);
          }
        }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[m][nt][e] = keep * S[m][nt][e] + acc[m][nt][e] * f0 * f1;
    }
  }
  float* out = cr.work + ((int64_t)seg * c.B * c.H + bh) * ((int64_t)dk * p.dv) + v0;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * (w + 4 * m) + g + (e >> 1) * 8, j = 8 * (nt0 + nt) + t2 + (e & 1);
        if (i < dk && j < dv) out[(int64_t)i * p.dv + j] = S[m][nt][e];
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
  const float full = la_power32(l, seg_tokens);
  for (int s0 = 0; s0 < segments; s0 += 4) {
    float add[4];
    float* at = cr.work + ((int64_t)s0 * c.B * c.H + bh) * states + e;
    const int64_t step = (int64_t)c.B * c.H * states;
#pragma unroll
    for (int i = 0; i < 4; ++i) add[i] = s0 + i < segments ? at[i * step] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i;
      if (s >= segments) break;
      at[i * step] = S;
      const int64_t left = (int64_t)n - (int64_t)s * seg_tokens;
      const int count = (int)(left < 0 ? 0 : left < seg_tokens ? left : seg_tokens);
      const int times = (p.reverse && s == 0 && count > 0) ? count - 1 : count;
      const float f = times == 0 ? 1.f : times == seg_tokens ? full : la_power32(l, times);
      if (count > 0) S = f * S + add[i];
    }
  }
  if (p.s_out) p.s_out[bh * states + e] = (p.reverse && n > 0) ? (float)l * S : S;
}

// Segments for `blocks` blocks of one segment: as many as use the resident blocks of the GPU best, where
// the main pass costs its chunks, the state pass 0.4 of that (165 us beside 435), and a segment's state about three chunks to
// write, hand through and read.  Measured with the number of segments forced, forward / gradients in us:
//   8192 x 2 x 16 heads of 128    1: 1101 / 1718    2: 785 / 2041    4: 617 / 1646    8: 641 / 1660     taken: 617 / 1552
//   8192 x 8 heads of 64          1: 723 / 727      4: 241 / 251     12: 90 / 149     16: 69 / 132      taken: 68 / 133
//   2000 x 4 heads of 128         1: 269 / 269      4: 104 / 106     12: 48 / 74      16: 38 / 87       taken: 38 / 74
//   700 x 4 x 8 heads of 64       1: 63 / 63        2: 53 / 83       4: 31 / 56       8: 36 / 70        taken: 31 / 56
//   1999 x 6 x 12 of 48 and 80    1: 171 / 474      2: 197 / 587     3: 186 / 607     4: 212 / 571      taken: 186 / 474
//   the same, ragged              1: 226 / 423      2: 199 / 518     3: 169 / 531     8: 177 / 530      taken: 171 / 421
static int lc_segments(int64_t T, int64_t blocks, int resident) {
  const int64_t chunks = ceil_div(T, LC);
  int best = 1;
  double best_cost = (double)chunks * (double)ceil_div(blocks, resident);
  for (int s = 2; s <= 64 && 2 * s <= chunks; ++s) {
    const int64_t per = ceil_div(chunks, s);
    const double cost = (1.4 * (double)per + 3.0) * (double)ceil_div(blocks * s, resident);
    if (cost < best_cost) {
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
  // no more blocks than SMs: eight warps a block (24 tokens of 8 heads of 64: 10.2 -> 8.2 us; more blocks share the SMs better
  // with four, 100 x 128 x 16 heads: 469 us against 518 then)
  const bool few = blocks * count <= b200::state().sm_count;
  auto main_kernel = few ? (vec ? la_chunk_kernel<DK, 256, true> : la_chunk_kernel<DK, 256, false>)
                         : (vec ? la_chunk_kernel<DK, 128, true> : la_chunk_kernel<DK, 128, false>);
  B200_CUDA(cudaFuncSetAttribute(main_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if (p.segments > 1) {
    auto state_kernel = vec ? la_state_kernel<DK, true> : la_state_kernel<DK, false>;
    const size_t state_smem = (size_t)4 * LC * (DK + LC_COLS);       // both parts of k and v
    B200_CUDA(cudaFuncSetAttribute(state_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)state_smem));
    state_kernel<<<dim3((unsigned)blocks, (unsigned)count), LS_THREADS, state_smem, st>>>(c, all, p.segments, p.seg_tokens, p.slabs);
    B200_LAUNCH_CHECK();
    const int64_t most = (int64_t)all.run[0].r.dk * all.run[0].r.dv;      // the same product for every run
    la_segments_kernel<<<dim3((unsigned)ceil_div(most, 256), (unsigned)((int64_t)c.B * c.H), (unsigned)count), 256, 0, st>>>(c, all, p.segments, p.seg_tokens);
    B200_LAUNCH_CHECK();
  }
  main_kernel<<<dim3((unsigned)blocks, (unsigned)count), few ? 256 : 128, smem, st>>>(c, all, p.segments, p.seg_tokens, p.slabs, b200::state().sm_count);
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
    vec = vec && runs[i].dk % 4 == 0 && runs[i].dv % 4 == 0 && aligned16(runs[i].o) && aligned16(runs[i].s_in) && aligned16(runs[i].s_out) &&
          runs[i].os.t % 4 == 0 && runs[i].os.b % 4 == 0 && runs[i].os.h % 4 == 0;
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
