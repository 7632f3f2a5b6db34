// Decayed linear attention, recurrent form, for single tokens (the step of a model that answers) and short sequences:
// the state stays on the SM while the tokens pass by.
//
// Bound for a single token: HBM, the state is read once and written once (8 dk dv bytes) and everything else is small;
// the state, k, q and v are all asked for at once, and the registers are held to what lets six blocks of 128 threads
// share an SM (512 x 16 states of 128 x 128: 173 us on the device under the profiler, where five blocks took 184 and eight
// 189; a whole call 188 to 190; floor 166).  For several tokens: latency.
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "../../include/b200_handler.h"
#include "linear_attention.cuh"

namespace b200 {

struct LaRuns {
  LaRun run[3];
};

constexpr int LR_COLS = 32, LR_THREADS = 128;

__device__ __forceinline__ int64_t la_offset(const LaStrides& x, int b, int h) {
  return (int64_t)b * x.b + (int64_t)(x.div == 1 ? h : h / x.div) * x.h;
}

// 32 columns of the state of one (sequence, head), a slab, lie in the registers of `wps` warps (1, 2 or 4); columns never
// meet, so slabs are independent.  Lane: four columns cg (of 8 groups), rows R rl + r, r < R; dv is a multiple of 4 and
// states start on 16 bytes.  VEC: so do the rows of q, k and v, and dk is a multiple of 4.  ONE: a single token (the next
// token's registers are not needed).
template <int R, bool VEC, bool ONE>
__global__ void __launch_bounds__(LR_THREADS, R == 8 ? (ONE ? 6 : 5) : 8) la_recurrent_kernel(LaCommon c, LaRuns runs, int max_slabs, int wps) {
  __shared__ __align__(16) float part[2][4][LR_COLS];      // written as float4
  const LaRun& p = runs.run[blockIdx.y];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned group = (unsigned)warp / wps, id = blockIdx.x * (4u / wps) + group;
  const unsigned bh = id / (unsigned)max_slabs;
  const int c0 = (int)(id - bh * max_slabs) * LR_COLS;
  const int dk = p.dk, dv = p.dv;
  if (bh >= (unsigned)c.B * (unsigned)c.H || c0 >= dv) return;
  const int b = (int)(bh / (unsigned)c.H), h = (int)bh - b * c.H;
  const int n = la_length(c, b);
  const float l = c.decay[h];
  const int cg = lane & 7, rl = (warp - group * wps) * 4 + (lane >> 3);
  const int64_t tok0 = p.reverse ? n - 1 : 0, dir = p.reverse ? -1 : 1;
  const float *q = p.q + la_offset(p.qs, b, h) + tok0 * p.qs.t, *k = p.k + la_offset(p.ks, b, h) + tok0 * p.ks.t,
              *v = p.v + la_offset(p.vs, b, h) + tok0 * p.vs.t;
  float* o = p.o + la_offset(p.os, b, h);
  const int col = c0 + 4 * cg;
  auto meet = [&]() {       // the warps of this slab
    if (wps == 1) __syncwarp();
    else if (group == 0) asm volatile("bar.sync 1, %0;" ::"r"(32 * wps) : "memory");
    else asm volatile("bar.sync 2, %0;" ::"r"(32 * wps) : "memory");
  };

  float S[R][4], kk[R], qq[R], vv[4];
  const float* s_in = p.s_in ? p.s_in + (int64_t)bh * dk * dv : nullptr;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = R * rl + r;
#pragma unroll
    for (int j = 0; j < 4; ++j) S[r][j] = 0.f;
    if (!s_in || i >= dk || col >= dv) continue;
    if (!p.s_in_t) {
      const float4 x = *reinterpret_cast<const float4*>(s_in + (int64_t)i * dv + col);
      S[r][0] = x.x; S[r][1] = x.y; S[r][2] = x.z; S[r][3] = x.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) S[r][j] = s_in[(int64_t)(col + j) * dk + i];
    }
  }
  auto fetch = [&](int step) {
    const float *qt = q + dir * step * p.qs.t, *kt = k + dir * step * p.ks.t, *vt = v + dir * step * p.vs.t;
    const int i = R * rl;
    if (VEC) {
      using V = typename std::conditional<R == 2, float2, float4>::type;
      constexpr int W = R == 2 ? 2 : 4;
#pragma unroll
      for (int r = 0; r < R; r += W) {        // dk is a multiple of 4: a vector is inside or outside as a whole
        V a = {}, x = {};
        if (i + r < dk) {
          a = *reinterpret_cast<const V*>(qt + i + r);
          x = *reinterpret_cast<const V*>(kt + i + r);
        }
        memcpy(qq + r, &a, sizeof(V));
        memcpy(kk + r, &x, sizeof(V));
      }
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col < dv) x = *reinterpret_cast<const float4*>(vt + col);
      memcpy(vv, &x, sizeof(x));
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        qq[r] = i + r < dk ? qt[i + r] : 0.f;
        kk[r] = i + r < dk ? kt[i + r] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) vv[j] = col < dv ? vt[col + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) vv[j] *= p.k_scale;
  };
  auto store_state = [&](float f) {
    if (!p.s_out || col >= dv) return;
    float* s = p.s_out + (int64_t)bh * dk * dv;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = R * rl + r;
      if (i < dk) *reinterpret_cast<float4*>(s + (int64_t)i * dv + col) = make_float4(f * S[r][0], f * S[r][1], f * S[r][2], f * S[r][3]);
    }
  };
  if (n > 0) fetch(0);
  for (int step = 0; step < (ONE ? min(n, 1) : n); ++step) {
    const float f = (p.reverse && step == 0) ? 1.f : l;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        S[r][j] = f * S[r][j] + kk[r] * vv[j];
        acc[j] += qq[r] * S[r][j];
      }
    if (!ONE && step + 1 < n) fetch(step + 1);
    else store_state(p.reverse ? l : 1.f);
#pragma unroll
    for (int m = 8; m < 32; m <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], m);
    if (lane < 8) *reinterpret_cast<float4*>(&part[step & 1][warp][4 * cg]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    meet();      // the sums of this step are in place; those of the step before have been read
    if (warp == (int)group * wps && c0 + lane < dv) {
      float x = part[step & 1][warp][lane];
      for (int u = 1; u < wps; ++u) x += part[step & 1][warp + u][lane];
      x *= p.o_scale;
      float* dst = o + (tok0 + dir * step) * p.os.t + c0 + lane;
      *dst = p.accumulate ? *dst + x : x;
    }
  }
  if (!p.accumulate && warp == (int)group * wps && c0 + lane < dv)      // tokens behind the end of the sequence
    for (int64_t t = n; t < c.T; ++t) o[t * p.os.t + c0 + lane] = 0.f;
  if (n == 0) store_state(1.f);
}

// Any dv and any alignment: a block for the state of one (sequence, head), 32 bits a lane.  Thread: column j, rows
// rg + groups * r, r < R, in registers.
template <int R>
__global__ void __launch_bounds__(1024, R <= 8 ? 2 : 1) la_recurrent_any_kernel(LaCommon c, LaRuns runs, int cols_log2) {
  __shared__ float qkv[3 * LA_MAX_DIM];
  extern __shared__ float part[];
  const LaRun& p = runs.run[blockIdx.y];
  const int bh = blockIdx.x, b = bh / c.H, h = bh - b * c.H;
  const int n = la_length(c, b), dk = p.dk, dv = p.dv, tid = threadIdx.x, threads = blockDim.x;
  const float l = c.decay[h];
  const int64_t tok0 = p.reverse ? n - 1 : 0, dir = p.reverse ? -1 : 1;
  const float *q = p.q + la_offset(p.qs, b, h) + tok0 * p.qs.t, *k = p.k + la_offset(p.ks, b, h) + tok0 * p.ks.t,
              *v = p.v + la_offset(p.vs, b, h) + tok0 * p.vs.t;
  float* o = p.o + la_offset(p.os, b, h);
  const int cols = 1 << cols_log2, j = tid & (cols - 1), rg = tid >> cols_log2, groups = threads >> cols_log2;
  const int64_t state = (int64_t)bh * dk * dv;
  float S[R];
#pragma unroll
  for (int r = 0; r < R; ++r) S[r] = 0.f;
  if (p.s_in && j < dv) {
    const float* s = p.s_in + state + (p.s_in_t ? j * dk + rg : rg * dv + j);
    const int next = groups * (p.s_in_t ? 1 : dv);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (rg + groups * r < dk) S[r] = s[r * next];
  }
  for (int step = 0; step < n; ++step) {
    const float *qt = q + dir * step * p.qs.t, *kt = k + dir * step * p.ks.t, *vt = v + dir * step * p.vs.t;
    for (int i = tid; i < dk; i += threads) {
      qkv[i] = qt[i];
      qkv[LA_MAX_DIM + i] = kt[i] * p.k_scale;
    }
    for (int i = tid; i < dv; i += threads) qkv[2 * LA_MAX_DIM + i] = vt[i];
    __syncthreads();
    const float f = (p.reverse && step == 0) ? 1.f : l, vj = j < dv ? qkv[2 * LA_MAX_DIM + j] : 0.f;
    float acc = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = min(rg + groups * r, LA_MAX_DIM - 1);
      if (rg + groups * r < dk) {
        S[r] = f * S[r] + qkv[LA_MAX_DIM + i] * vj;
        acc += qkv[i] * S[r];
      }
    }
    part[tid] = acc;
    __syncthreads();
    if (tid < dv) {
      float x = part[tid];
      for (int u = 1; u < groups; ++u) x += part[(u << cols_log2) + tid];
      x *= p.o_scale;
      float* dst = o + (tok0 + dir * step) * p.os.t + tid;
      *dst = p.accumulate ? *dst + x : x;
    }
  }
  if (!p.accumulate)       // tokens behind the end of the sequence
    for (int64_t t = n; t < c.T; ++t)
      for (int i = tid; i < dv; i += threads) o[t * p.os.t + i] = 0.f;
  if (p.s_out && j < dv) {
    const float f = (p.reverse && n > 0) ? l : 1.f;
    float* s = p.s_out + state + rg * dv + j;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (rg + groups * r < dk) s[r * groups * dv] = f * S[r];
  }
}

// One token for many states of any dv and alignment.  The states of consecutive (sequence, head)s are one run of memory: a
// block takes `per` of them into shared memory as they lie, 128 bits at a time counted from the boundary before the first,
// works on them there column by column, and writes them back the same way.  k and q lie beside them, padded to four
// rows, so that a thread reads four rows' factors at once.
// Bound: HBM (512 x 16 states of 127 x 126: 380 us by 32-bit accesses from the columns in registers, 223 here, floor
// 163; 4000 x 4 of 90 x 97: 642 and 238, floor 174; 2182 x 16 of 52 x 15: 97 and 64, floor 36).
struct LaFlatState {
  const float *q, *k, *v;
  float* o;
  float decay;
  int live;
};
constexpr int LF_THREADS = 256, LF_MOST = 64;

__host__ __device__ __forceinline__ int lf_rows(int dk) { return (dk + 3) & ~3; }

__global__ void __launch_bounds__(LF_THREADS) la_flat_step_kernel(LaCommon c, LaRun p, int per, int cols_log2) {
  extern __shared__ __align__(16) float lf_smem[];
  __shared__ LaFlatState one[LF_MOST];
  __shared__ float part[LF_THREADS];
  const int dk = p.dk, dv = p.dv, N = dk * dv, dkp = lf_rows(dk), tid = threadIdx.x, threads = blockDim.x;
  const int64_t BH = (int64_t)c.B * c.H, bh0 = (int64_t)blockIdx.x * per;
  const int count = (int)min((int64_t)per, BH - bh0), total = count * N;
  float* kq = lf_smem;                                       // k and q of each state
  float* vs = kq + 2 * per * dkp;                            // v of each state
  const float* s_in = p.s_in + bh0 * N;
  float* s_out = p.s_out + bh0 * N;
  const int off = (int)((reinterpret_cast<uintptr_t>(s_in) >> 2) & 3);
  float* S = vs + ((per * dv + 3) & ~3) + off;               // element e of the run at S[e]
  // ---- the states on their way
  const int head = min(total, (4 - off) & 3), whole = (total - head) >> 2, tail = head + 4 * whole;
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(S);
  for (int i = tid; i < whole; i += threads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 4 * (head + 4 * i)), "l"(s_in + head + 4 * i) : "memory");
  if (tid < head) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * tid), "l"(s_in + tid) : "memory");
  if (tail + tid < total) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + 4 * (tail + tid)), "l"(s_in + tail + tid) : "memory");
  // ---- the rest of them
  if (tid < count) {
    const int bh = (int)(bh0 + tid), b = bh / c.H, h = bh - b * c.H;
    one[tid] = {p.q + la_offset(p.qs, b, h), p.k + la_offset(p.ks, b, h), p.v + la_offset(p.vs, b, h), p.o + la_offset(p.os, b, h), c.decay[h],
                la_length(c, b) > 0};
  }
  __syncthreads();
  for (int i = tid; i < count * dkp; i += threads) {
    const int g = i / dkp, row = i - g * dkp;
    const bool in = row < dk && one[g].live;
    kq[2 * g * dkp + row] = in ? one[g].k[row] * p.k_scale : 0.f;
    kq[(2 * g + 1) * dkp + row] = in ? one[g].q[row] : 0.f;
  }
  for (int i = tid; i < count * dv; i += threads) {
    const int g = i / dv;
    vs[i] = one[g].live ? one[g].v[i - g * dv] : 0.f;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // ---- thread: a column of a state, a share of the rows
  const int cols = 1 << cols_log2, groups = threads >> cols_log2, rg = tid >> cols_log2;
  const int rows = lf_rows((dk + groups - 1) / groups), first = rg * rows, last = min(dk, first + rows);
  for (int c0 = 0; c0 < count * dv; c0 += cols) {            // one pass when there are groups
    const int col = c0 + (tid & (cols - 1));
    const int g = min(col / dv, count - 1), j = col - g * dv;
    float acc = 0.f;
    if (col < count * dv && one[g].live) {
      const float l = one[g].decay, vj = vs[col];
      const float4* kk = reinterpret_cast<const float4*>(kq + 2 * g * dkp);
      const float4* qq = reinterpret_cast<const float4*>(kq + (2 * g + 1) * dkp);
      float* s = S + g * N + j;
      for (int i = first; i < last; i += 4) {
        const float4 k4 = kk[i >> 2], q4 = qq[i >> 2];
        const float kx[4] = {k4.x, k4.y, k4.z, k4.w}, qx[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u < last) {
            const float x = l * s[(i + u) * dv] + kx[u] * vj;
            s[(i + u) * dv] = x;
            acc += qx[u] * x;
          }
      }
    }
    if (groups > 1) {
      part[tid] = acc;
      __syncthreads();
      if (rg == 0)
        for (int u = 1; u < groups; ++u) acc += part[tid + (u << cols_log2)];
    }
    if (rg == 0 && col < count * dv) one[g].o[j] = one[g].live ? p.o_scale * acc : 0.f;
  }
  __syncthreads();
  // ---- back
  if (((reinterpret_cast<uintptr_t>(s_out) >> 2) & 3) == off) {
    for (int i = tid; i < whole; i += threads) *reinterpret_cast<float4*>(s_out + head + 4 * i) = *reinterpret_cast<const float4*>(S + head + 4 * i);
    if (tid < head) s_out[tid] = S[tid];
    if (tail + tid < total) s_out[tail + tid] = S[tail + tid];
  } else {
    for (int i = tid; i < total; i += threads) s_out[i] = S[i];
  }
}

// Floats of shared memory for `per` states.
static int64_t lf_floats(int per, int dk, int dv) { return (int64_t)per * (2 * lf_rows(dk) + (int64_t)dk * dv) + (((int64_t)per * dv + 3) & ~3ll) + 4; }

static int la_flat_step(const LaCommon& c, const LaRun& run) {
  const int64_t BH = (int64_t)c.B * c.H;
  // 128 threads with at most 20 KiB (2000 x 8 states of 64 x 63: 104 us, 256 with 40 KiB 110) or, for states of more than 16 KiB, 256
  // (512 x 16 of 127 x 126: 223 us, 128 threads 246); one state at least, eight blocks for each SM at least
  const int threads = run.dk * run.dv <= 4096 ? 128 : LF_THREADS;
  int per = 1;
  while (per < LF_MOST && lf_floats(per + 1, run.dk, run.dv) <= 40 * threads && ceil_div(BH, per + 1) >= 8ll * state().sm_count) ++per;
  int log2 = 5;
  while ((1 << log2) < threads && (1 << log2) < per * run.dv) ++log2;
  const int64_t smem = lf_floats(per, run.dk, run.dv) * 4;
  static bool ready = false;
  if (!ready) {
    B200_CUDA(cudaFuncSetAttribute(la_flat_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)lf_floats(1, LA_MAX_DIM, LA_MAX_DIM) * 4));
    ready = true;
  }
  la_flat_step_kernel<<<(unsigned)ceil_div(BH, per), threads, smem, state().stream>>>(c, run, per, log2);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

// One launch for up to three runs over the same sequences.
int la_recurrent(const LaCommon& c, const LaRun* runs, int count) {
  LaRuns all = {};
  int dk = 0, dv = 0;
  bool whole = true, vec = true;
  for (int i = 0; i < count; ++i) {
    all.run[i] = runs[i];
    dk = std::max(dk, runs[i].dk);
    dv = std::max(dv, runs[i].dv);
    whole = whole && runs[i].dv % 4 == 0 && aligned16(runs[i].s_in) && aligned16(runs[i].s_out);
    vec = vec && runs[i].dk % 4 == 0;
    for (const float* a : {runs[i].q, runs[i].k, runs[i].v}) vec = vec && aligned16(a);
    for (const LaStrides* x : {&runs[i].qs, &runs[i].ks, &runs[i].vs}) vec = vec && x->t % 4 == 0 && x->b % 4 == 0 && x->h % 4 == 0;
  }
  const int64_t BH = (int64_t)c.B * c.H;
  const cudaStream_t st = state().stream;
  // (64 x 8 states of 40 x 75: 11.1 us by columns, 7.0 flat; 100 x 4 of 30 x 50: 4.9 and 5.6)
  if (!whole && c.T == 1 && count == 1 && runs[0].s_in && runs[0].s_out && BH >= 3ll * b200::state().sm_count) return la_flat_step(c, runs[0]);
  if (!whole) {
    int log2 = 3, threads = 128;
    while ((1 << log2) < dv) ++log2;
    while ((int64_t)dk << log2 > 16ll * threads) threads *= 2;      // 1024 at dk = dv = 128
    const int rows = (int)ceil_div(dk, threads >> log2);
    auto kernel = rows <= 4 ? la_recurrent_any_kernel<4> : rows <= 8 ? la_recurrent_any_kernel<8> : la_recurrent_any_kernel<16>;
    kernel<<<dim3((unsigned)BH, (unsigned)count), threads, threads * sizeof(float), st>>>(c, all, log2);
    B200_LAUNCH_CHECK();
    return B200_OK;
  }
  const int slabs = (int)ceil_div(dv, LR_COLS);
  B200_REQUIRE(BH * slabs < (1ll << 31), "linear attention: extent too large");
  // Few slabs: four warps each, for the latency.  Many: as few as hold it with eight rows (dk up to 16: four) a lane, for
  // the loads in flight.
  int rows, wps;
  if (BH * slabs * count <= 4ll * state().sm_count) {
    wps = 4;
    rows = dk <= 32 ? 2 : dk <= 64 ? 4 : 8;
  } else {
    rows = dk <= 16 ? 4 : 8;
    wps = dk <= 32 ? 1 : dk <= 64 ? 2 : 4;
  }
#define LR_KERNELS(R)                                                                                  \
  (c.T == 1 ? (vec ? la_recurrent_kernel<R, true, true> : la_recurrent_kernel<R, false, true>)         \
            : (vec ? la_recurrent_kernel<R, true, false> : la_recurrent_kernel<R, false, false>))
  auto kernel = rows == 2 ? LR_KERNELS(2) : rows == 4 ? LR_KERNELS(4) : LR_KERNELS(8);
#undef LR_KERNELS
  kernel<<<dim3((unsigned)ceil_div(BH * slabs, 4 / wps), (unsigned)count), LR_THREADS, 0, st>>>(c, all, slabs, wps);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

// dst (T, B, heads, d) (+)= the sum over the `group` operator heads that share a head, in order; src is
// (T, B, heads * group, d), contiguous.
__global__ void __launch_bounds__(256) la_share_kernel(const float* src, float* dst, LaStrides ds, int64_t rows, int B, int heads, int group,
                                                       int d, int accumulate) {
  const int64_t total = rows * heads * d;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int e = (int)(i % d);
    const int64_t rh = i / d;
    const int h = (int)(rh % heads);
    const int64_t row = rh / heads, t = row / B, b = row % B;
    const float* s = src + ((row * heads + h) * group) * d + e;
    float sum = s[0];
    for (int g = 1; g < group; ++g) sum += s[(int64_t)g * d];
    float* o = dst + t * ds.t + b * ds.b + h * ds.h + e;
    *o = accumulate ? *o + sum : sum;
  }
}

// Sequences of up to this many tokens take the recurrent form.  Its time grows with the tokens, that of a chunk hardly does; they meet
// at 6 to 11 tokens (forward / gradients in us on the device, recurrent against chunked):
//   tokens, 8 heads of 64            4: 5.3 / 5.2, 6.4 / 6.3       8: 8.1 / 8.1, 6.5 / 6.3        12: 10.9 / 10.8, 6.7 / 6.5
//   128 x 16 heads of 64             4: 22 / 68, 46 / 126          8: 38 / 110, 47 / 127          12: 54 / 154, 49 / 133
//   64 x 16 heads of 128             4: 51 / 133, 93 / 262         8: 79 / 212, 94 / 267          12: 108 / 292, 97 / 276
//   64 x 8 heads over 2, 40 and 75   4: 19 / 112, 27 / 87          8: 31 / 185, 27 / 87           12: 44 / 260, 29 / 93
constexpr int LA_RECURRENT_TOKENS = 8;

static int la_run(const LaCommon& c, const LaRun* runs, int count, float* work) {
  return c.T <= LA_RECURRENT_TOKENS ? la_recurrent(c, runs, count) : la_chunked(c, runs, count, work);
}

static int la_check(const char* what, int64_t T, int64_t B, int64_t H, int64_t kv_heads, int64_t dk, int64_t dv) {
  B200_REQUIRE(T >= 0 && B >= 0 && H >= 0 && kv_heads >= 0 && dk >= 0 && dv >= 0, "%s: negative extent", what);
  B200_REQUIRE(B * H == 0 || (dk > 0 && dv > 0), "%s: heads without values", what);
  B200_REQUIRE(dk <= LA_MAX_DIM && dv <= LA_MAX_DIM, "%s: heads of more than %d values are not supported", what, LA_MAX_DIM);
  B200_REQUIRE(T < (1ll << 31) && B * H < (1ll << 31), "%s: extent exceeds 2^31", what);
  B200_REQUIRE(H == 0 || (kv_heads > 0 && H % kv_heads == 0), "%s: %lld heads cannot share %lld key/value heads", what, (long long)H,
               (long long)kv_heads);
  return B200_OK;
}
// t, b and head strides of array i; NULL: all arrays are contiguous
static LaStrides la_strides(const int64_t* s, int i, int64_t div, int64_t B, int64_t heads, int64_t d) {
  if (!s) return LaStrides{B * heads * d, heads * d, d, (int)div};
  return LaStrides{s[3 * i], s[3 * i + 1], s[3 * i + 2], (int)div};
}

}  // namespace b200

using namespace b200;

B200_API int64_t b200_linear_attention_forward_scratch_floats(int64_t T, int64_t B, int64_t H, int64_t dk, int64_t dv) {
  if (T <= LA_RECURRENT_TOKENS || B * H <= 0 || dk <= 0 || dv <= 0 || dk > LA_MAX_DIM || dv > LA_MAX_DIM) return 0;
  return la_chunked_work(T, B * H, (int)dk, (int)dv, false);
}

B200_API int b200_linear_attention_forward(const b200_linear_attention_args* args) {
  if (int rc = require_ready()) return rc;
  B200_REQUIRE(args, "linear attention: NULL arguments");
  const auto& [q, k, v, decay, out, state, state_out, lengths, strides, scratch, scratch_floats, T, B, H, kv_heads, dk, dv, scale] = *args;
  if (int rc = la_check("linear attention", T, B, H, kv_heads, dk, dv)) return rc;
  if (B * H == 0) return B200_OK;
  B200_REQUIRE(scratch_floats >= b200_linear_attention_forward_scratch_floats(T, B, H, dk, dv), "linear attention: scratch too small");
  B200_REQUIRE(decay && (T == 0 || (q && k && v && out)), "linear attention: NULL operand");
  const int64_t g = H / kv_heads;
  const int64_t* s = strides;
  LaCommon c = {decay, lengths, (int)T, (int)B, (int)H};
  LaRun r = {q, k, v, out, la_strides(s, 0, 1, B, H, dk), la_strides(s, 1, g, B, kv_heads, dk), la_strides(s, 2, g, B, kv_heads, dv),
             la_strides(s, 3, 1, B, H, dv), state, state_out, 0, 0,
             0, (int)dk, (int)dv, 1.f, scale};
  return la_run(c, &r, 1, scratch);
}

B200_API int64_t b200_linear_attention_backward_scratch_floats(int64_t T, int64_t B, int64_t H, int64_t kv_heads, int64_t dk, int64_t dv) {
  if (T <= 0 || B * H <= 0 || dk <= 0 || dv <= 0 || dk > LA_MAX_DIM || dv > LA_MAX_DIM) return 0;
  return (kv_heads < H ? T * B * H * (dk + dv) : 0) + (T <= LA_RECURRENT_TOKENS ? 0 : la_chunked_work(T, B * H, (int)dk, (int)dv, true));
}

B200_API int b200_linear_attention_backward(const float* q, const float* k, const float* v, const float* decay, const float* dout, float* dq,
                                            float* dk_out, float* dv_out, const float* state, const float* dstate_out, float* dstate,
                                            const float* lengths, int64_t T, int64_t B, int64_t H, int64_t kv_heads, int64_t dk, int64_t dv,
                                            const int64_t* strides, float scale, int accumulate, float* scratch, int64_t scratch_floats) {
  if (int rc = require_ready()) return rc;
  if (int rc = la_check("linear attention", T, B, H, kv_heads, dk, dv)) return rc;
  if (B * H == 0) return B200_OK;
  B200_REQUIRE(decay && (T == 0 || (q && k && v && dout && dq && dk_out && dv_out)), "linear attention: NULL operand");
  B200_REQUIRE(scratch_floats >= b200_linear_attention_backward_scratch_floats(T, B, H, kv_heads, dk, dv), "linear attention: scratch too small");
  B200_REQUIRE(!dstate || dstate != dstate_out, "linear attention: dstate overlaps dstate_out");   // two gradients read it
  const int64_t g = H / kv_heads;
  const int64_t* s = strides;
  const int acc = accumulate ? 1 : 0;
  LaCommon c = {decay, lengths, (int)T, (int)B, (int)H};
  const LaStrides qs = la_strides(s, 0, 1, B, H, dk), ks = la_strides(s, 1, g, B, kv_heads, dk), vs = la_strides(s, 2, g, B, kv_heads, dv),
                  dos = la_strides(s, 3, 1, B, H, dv), dqs = la_strides(s, 4, 1, B, H, dk);
  const LaStrides shared[2] = {la_strides(s, 5, 1, B, kv_heads, dk), la_strides(s, 6, 1, B, kv_heads, dv)};
  LaStrides dks = shared[0], dvs = shared[1];
  float *dk_w = dk_out, *dv_w = dv_out;
  if (g > 1) {     // one gradient for each head of q first, then the sum over the heads that share
    dk_w = scratch;
    dv_w = scratch + T * B * H * dk;
    dks = LaStrides{B * H * dk, H * dk, dk, 1};
    dvs = LaStrides{B * H * dv, H * dv, dv, 1};
  }
  LaRun runs[3] = {
      {dout, v, k, dq, dos, vs, ks, dqs, state, nullptr, 1, 0, acc, (int)dv, (int)dk, 1.f, scale},
      {v, dout, q, dk_w, vs, dos, qs, dks, dstate_out, nullptr, 1, 1, g > 1 ? 0 : acc, (int)dv, (int)dk, scale, 1.f},
      {k, q, dout, dv_w, ks, qs, dos, dvs, dstate_out, dstate, 0, 1, g > 1 ? 0 : acc, (int)dk, (int)dv, scale, 1.f},
  };
  if (int rc = la_run(c, runs, 3, scratch + (g > 1 ? T * B * H * (dk + dv) : 0))) return rc;
  if (g > 1 && T > 0) {
    for (int i = 0; i < 2; ++i) {
      const int d = (int)(i ? dv : dk);
      const int64_t total = T * B * kv_heads * d;
      const int64_t blocks = std::min<int64_t>(ceil_div(total, 256), (int64_t)b200::state().sm_count * 16);
      la_share_kernel<<<(unsigned)blocks, 256, 0, b200::state().stream>>>(i ? dv_w : dk_w, i ? dv_out : dk_out, shared[i], T * B,
                                                                          (int)B, (int)kv_heads, (int)g, d, acc);
      B200_LAUNCH_CHECK();
    }
  }
  return B200_OK;
}
