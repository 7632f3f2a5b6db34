// out = alpha a b^T + beta add in fp32 accuracy on tcgen05.mma kind::f16, for operands that are already split
// into two half-precision planes (hi = fp16(x), lo = fp16(x - hi), 22 bits together): what the Newton-Schulz
// iteration of muon.cu multiplies.  Its matrices stay below 3 in magnitude, so one fixed scale keeps them in
// the range of half precision, and the epilogue of one product writes the planes the next one reads: nothing
// is split inside the main loop.
//
//  * a b = hi.hi + hi.lo + lo.hi: three MMAs for each 128 x BN x 16 step, at twice the rate and half the operand
//    bytes of three TF32 MMAs of depth 8.
//  * The tensor core truncates when it adds into its accumulator.  Each k-block of 64 is therefore a chunk of
//    its own: its eight small products first, while the accumulator is small, then its four large ones; the
//    finished chunk is added to fp32 registers with rounding while the next runs in the other half of tensor
//    memory.
//  * Roles (320 threads): warp 0 TMA, warp 1 MMA and tensor memory, warps 2 to 9 drain and epilogue (a lane owns
//    a row; two groups of four warps own half the columns each).
//  * The transpose leaves straight from the registers: 32 lanes hold 32 rows of a column; neighbouring lanes
//    trade halves so that each stores 32 bits.
//  * A symmetric product computes the tiles that reach the upper triangle; an element above the diagonal is
//    stored at both places, so the result is symmetric bit for bit.
//  * Every wait is bounded, as in the general GEMM.
#include <cuda.h>

#include <algorithm>

#include "ns_gemm.cuh"
#include "tc_ptx.cuh"

namespace b200 {

int* device_error_flag();       // gemm_tc.cu

constexpr int NS_BM = 128, NS_BK = 64, NS_THREADS = 320;

template <int BN>
struct NsConfig {
  static constexpr int A_BYTES = NS_BM * NS_BK * 2, B_BYTES = BN * NS_BK * 2;      // one plane
  static constexpr int STAGE_BYTES = 2 * (A_BYTES + B_BYTES);
  static constexpr int STAGES = BN == 256 ? 2 : BN == 128 ? 3 : 4;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int ACC = BN / 2;                                                // columns of a drain group
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
};

struct NsEpilogue {
  const __half* add;            // NULL or planes like out's
  __half *out, *out_t;
  int ld_add, ld_out, ld_out_t;
  float alpha, beta;
};

// Tile t of the walk: bands of 8 row tiles, column by column inside a band, so that the blocks that run
// together share rows of both operands in L2.  Symmetric: only tiles that reach the diagonal or lie above it.
__device__ __forceinline__ bool ns_tile(int t, int tiles_m, int tiles_n, int bn, bool symmetric, int* i, int* j) {
  for (int band = 0; band < tiles_m; band += 8) {
    const int rows = min(8, tiles_m - band);
    for (int c = symmetric ? band * NS_BM / bn : 0; c < tiles_n; ++c) {
      // rows of this band whose tile at column c reaches the diagonal: 128 i <= bn (c + 1) - 1
      const int fit = symmetric ? min(rows, (bn * (c + 1) - 1) / NS_BM - band + 1) : rows;
      if (!symmetric) {         // all columns of the band alike
        if (t >= rows * tiles_n) break;
        *i = band + t % rows;
        *j = t / rows;
        return true;
      }
      if (t < fit) {
        *i = band + t;
        *j = c;
        return true;
      }
      t -= fit;
    }
    if (!symmetric) t -= rows * tiles_n;
  }
  return false;
}
static int ns_tiles(int tiles_m, int tiles_n, int bn, bool symmetric) {
  if (!symmetric) return tiles_m * tiles_n;
  int n = 0;
  for (int band = 0; band < tiles_m; band += 8) {
    const int rows = std::min(8, tiles_m - band);
    for (int c = band * NS_BM / bn; c < tiles_n; ++c) n += std::min(rows, (bn * (c + 1) - 1) / NS_BM - band + 1);
  }
  return n;
}

__device__ __forceinline__ uint32_t ns_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// 32 columns of one row: from acc (row `row`, columns col ..) to the planes.
template <bool DIAGONAL>
__device__ __forceinline__ void ns_store(const float* acc, const NsEpilogue& e, int64_t plane, int64_t plane_t, int row, int col, int M, int N) {
  uint32_t hi[16], lo[16];
  const bool in = row < M;
  const float alpha = e.alpha / NS_SCALE;
#pragma unroll
  for (int c8 = 0; c8 < 4; ++c8) {
    float add[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (e.add && in && col + 8 * c8 < e.ld_add) {
      const int64_t at = (int64_t)row * e.ld_add + col + 8 * c8;
      const uint4 h = *reinterpret_cast<const uint4*>(e.add + at), l = *reinterpret_cast<const uint4*>(e.add + plane + at);
      const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hw[u])), b = __half22float2(*reinterpret_cast<const __half2*>(&lw[u]));
        add[2 * u] = a.x + b.x;
        add[2 * u + 1] = a.y + b.y;
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float x = alpha * acc[8 * c8 + 2 * u] + e.beta * add[2 * u], y = alpha * acc[8 * c8 + 2 * u + 1] + e.beta * add[2 * u + 1];
      const __half2 h = __floats2half2_rn(x, y);
      const float2 f = __half22float2(h);
      hi[4 * c8 + u] = ns_bits(h);
      lo[4 * c8 + u] = ns_bits(__floats2half2_rn(x - f.x, y - f.y));
    }
  }
  if (e.out && in) {
#pragma unroll
    for (int c8 = 0; c8 < 4; ++c8) {
      const int c = col + 8 * c8;
      if (c >= e.ld_out) continue;
      __half* at = e.out + (int64_t)row * e.ld_out + c;
      if (!DIAGONAL || c >= row) {
        *reinterpret_cast<uint4*>(at) = make_uint4(hi[4 * c8], hi[4 * c8 + 1], hi[4 * c8 + 2], hi[4 * c8 + 3]);
        *reinterpret_cast<uint4*>(at + plane) = make_uint4(lo[4 * c8], lo[4 * c8 + 1], lo[4 * c8 + 2], lo[4 * c8 + 3]);
      } else if (c + 7 >= row) {              // the group that the diagonal crosses in this row
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (c + u >= row) {
            reinterpret_cast<uint16_t*>(at)[u] = (uint16_t)(hi[4 * c8 + u / 2] >> (16 * (u & 1)));
            reinterpret_cast<uint16_t*>(at + plane)[u] = (uint16_t)(lo[4 * c8 + u / 2] >> (16 * (u & 1)));
          }
      }
    }
  }
  if (e.out_t) {
    const int odd = row & 1, r0 = row - odd;
#pragma unroll
    for (int u = 0; u < 16; ++u) {            // columns 2 u and 2 u + 1: the even lane takes the first, the odd one the second
      const uint32_t ph = __shfl_xor_sync(0xffffffffu, hi[u], 1), pl = __shfl_xor_sync(0xffffffffu, lo[u], 1);
      const uint32_t wh = odd ? __byte_perm(ph, hi[u], 0x7632) : __byte_perm(hi[u], ph, 0x5410);
      const uint32_t wl = odd ? __byte_perm(pl, lo[u], 0x7632) : __byte_perm(lo[u], pl, 0x5410);
      const int c = col + 2 * u + odd;
      if (c >= N || r0 >= M) continue;
      __half* at = e.out_t + (int64_t)c * e.ld_out_t + r0;
      if (!DIAGONAL || c > r0 + 1) {
        *reinterpret_cast<uint32_t*>(at) = wh;
        *reinterpret_cast<uint32_t*>(at + plane_t) = wl;
      } else if (c == r0 + 1) {               // the second row of the pair is the diagonal
        *reinterpret_cast<uint16_t*>(at) = (uint16_t)wh;
        *reinterpret_cast<uint16_t*>(at + plane_t) = (uint16_t)wl;
      }
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, NsEpilogue e, int M, int N, int K, int batch,
               int symmetric, int* error_flag) {
  using Cfg = NsConfig<BN>;
  constexpr int S = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * Cfg::STAGE_BYTES);
  // bars[0..S) full, [S..2S) empty, [2S..2S+2) chunk ready, [2S+2..2S+4) chunk drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  int ti = 0, tj = 0;
  ns_tile(blockIdx.x, (M + NS_BM - 1) / NS_BM, (N + BN - 1) / BN, BN, symmetric, &ti, &tj);
  const int m0 = ti * NS_BM, n0 = tj * BN;
  const int num_kb = (K + NS_BK - 1) / NS_BK;
  const uint32_t bar0 = smem_u32(bars), smem_base = smem_u32(smem);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto acc_full_bar = [&](int i) { return bar0 + 8u * (2 * S + i); };
  auto acc_empty_bar = [&](int i) { return bar0 + 8u * (2 * S + 2 + i); };
  auto a_at = [&](int s, int plane) { return smem_base + s * Cfg::STAGE_BYTES + plane * Cfg::A_BYTES; };
  auto b_at = [&](int s, int plane) { return smem_base + s * Cfg::STAGE_BYTES + 2 * Cfg::A_BYTES + plane * Cfg::B_BYTES; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full_bar(i), 1);
      mbar_init(acc_empty_bar(i), 256);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_launch_dependents();
  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_d = *tmem_slot;
  pdl_wait();       // operands and outputs belong to the kernel before until here

  if (warp == 0) {
    if (lane == 0) {
      asm volatile("fence.proxy.async;" ::: "memory");      // the planes were written by ordinary stores
      int issued = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        const int s = kb % S;
        if (!mbar_wait(empty_bar(s), ((kb / S) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(full_bar(s), Cfg::STAGE_BYTES);
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
          tma_load_3d(a_at(s, plane), &map_a, kb * NS_BK, m0, plane * batch + b, full_bar(s));
          tma_load_3d(b_at(s, plane), &map_b, kb * NS_BK, n0, plane * batch + b, full_bar(s));
        }
        issued = kb + 1;
      }
      if (*abort_flag) {        // copies already issued must land before shared memory is released
        for (int kb = issued > S ? issued - S : 0; kb < issued; ++kb)
          for (uint32_t it = 0; it < TC_SPIN_LIMIT && !mbar_try_wait(full_bar(kb % S), (kb / S) & 1); ++it) __nanosleep(64);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // D = F32, A = B = F16, both K-major, N >> 3, M >> 4
    const uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(NS_BM >> 4) << 24);
    bool ok = true;
    for (int kb = 0; kb < num_kb && ok; ++kb) {
      const int s = kb % S, buf = kb & 1;
      ok = mbar_wait(acc_empty_bar(buf), ((kb >> 1) & 1) ^ 1, abort_flag) && mbar_wait(full_bar(s), (kb / S) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (lane == 0) {
        const uint32_t d = tmem_d + (uint32_t)(buf * BN);
        auto desc = [&](uint32_t at, int k) { return smem_desc(at + 32 * k, 16, 1024, 2); };
#pragma unroll
        for (int k = 0; k < NS_BK / 16; ++k) {          // the small products first
          mma_f16(d, desc(a_at(s, 1), k), desc(b_at(s, 0), k), idesc, k > 0);
          mma_f16(d, desc(a_at(s, 0), k), desc(b_at(s, 1), k), idesc, 1);
        }
#pragma unroll
        for (int k = 0; k < NS_BK / 16; ++k) mma_f16(d, desc(a_at(s, 0), k), desc(b_at(s, 0), k), idesc, 1);
        mma_commit(empty_bar(s));
        mma_commit(acc_full_bar(buf));
      }
      __syncwarp();
    }
    __syncwarp();
  } else {
    const int q = warp & 3, group = (warp - 2) >> 2;    // tensor-memory lanes, columns of this warp
    const uint32_t lane_bits = (uint32_t)(q * 32) << 16;
    float acc[Cfg::ACC];
#pragma unroll
    for (int j = 0; j < Cfg::ACC; ++j) acc[j] = 0.f;
    bool ok = true;
    for (int kb = 0; kb < num_kb && ok; ++kb) {
      const int buf = kb & 1;
      ok = mbar_wait(acc_full_bar(buf), (kb >> 1) & 1, abort_flag);
      __syncwarp();
      if (!ok) break;
      tc_fence_after();
      drain_add<Cfg::ACC>(tmem_d + lane_bits + (uint32_t)(buf * BN + group * Cfg::ACC), acc);
      tc_fence_before();
      mbar_arrive(acc_empty_bar(buf));
    }
    if (ok) {
      const int row = m0 + q * 32 + lane;
      e.add += e.add ? (int64_t)b * M * e.ld_add : 0;
      e.out += e.out ? (int64_t)b * M * e.ld_out : 0;
      e.out_t += e.out_t ? (int64_t)b * N * e.ld_out_t : 0;
      const int64_t plane = (int64_t)batch * M * (e.out ? e.ld_out : e.ld_add), plane_t = (int64_t)batch * N * e.ld_out_t;
#pragma unroll
      for (int cc = 0; cc < Cfg::ACC / 32; ++cc) {
        const int col = n0 + group * Cfg::ACC + 32 * cc;
        if (symmetric && col < m0 + q * 32 + 32) ns_store<true>(acc + 32 * cc, e, plane, plane_t, row, col, M, N);
        else if (col < N) ns_store<false>(acc + 32 * cc, e, plane, plane_t, row, col, M, N);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_d, Cfg::TMEM_COLS);
  }
  if (threadIdx.x == 0 && *abort_flag && error_flag) *error_flag = 1;
}

typedef CUresult (*NsEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Both planes of a stack: K along the rows, rows, then plane and matrix; boxes of 64 x box_rows.
static int ns_map(const NsMatrix& a, int batch, int box_rows, CUtensorMap* out) {
  static NsEncodeFn encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    B200_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q));
    B200_REQUIRE(fn != nullptr && q == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled is unavailable");
    encode = (NsEncodeFn)fn;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)a.cols, (cuuint64_t)a.rows, (cuuint64_t)2 * batch};
  const cuuint64_t strides[2] = {(cuuint64_t)a.ld * 2, (cuuint64_t)a.ld * a.rows * 2};
  const cuuint32_t box[3] = {(cuuint32_t)NS_BK, (cuuint32_t)box_rows, 1u}, one[3] = {1u, 1u, 1u};
  const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return B200_OK;
}

template <int BN>
static int ns_launch(const NsMatrix& a, const NsMatrix& b, const NsEpilogue& e, int batch, bool symmetric) {
  CUtensorMap ma, mb;
  if (int rc = ns_map(a, batch, NS_BM, &ma)) return rc;
  if (int rc = ns_map(b, batch, BN, &mb)) return rc;
  int* flag = device_error_flag();
  B200_REQUIRE(flag != nullptr, "the device error flag cannot be set up");
  static bool ready = false;
  if (!ready) {
    B200_CUDA(cudaFuncSetAttribute(ns_gemm_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, NsConfig<BN>::SMEM_BYTES));
    ready = true;
  }
  const int tiles = ns_tiles((int)ceil_div(a.rows, NS_BM), (int)ceil_div(b.rows, BN), BN, symmetric);
  B200_CUDA(launch_maybe_pdl(true, ns_gemm_kernel<BN>, dim3((unsigned)tiles, (unsigned)batch), dim3(NS_THREADS), (size_t)NsConfig<BN>::SMEM_BYTES,
                             state().stream, ma, mb, e, a.rows, b.rows, a.cols, batch, symmetric ? 1 : 0, flag));
  B200_LAUNCH_CHECK();
  return B200_OK;
}

int ns_gemm(const NsMatrix& a, const NsMatrix& b, const NsMatrix* add, const NsMatrix* out, const NsMatrix* out_t, int batch, float alpha,
            float beta, bool symmetric) {
  NsEpilogue e = {add ? add->data : nullptr, out ? out->data : nullptr, out_t ? out_t->data : nullptr, add ? add->ld : 0, out ? out->ld : 0,
                  out_t ? out_t->ld : 0, alpha, beta};
  // the widest tile whose tiles still fill the GPU
  const int64_t tm = ceil_div(a.rows, NS_BM);
  const int sms = state().sm_count;
  if (batch * (int64_t)ns_tiles((int)tm, (int)ceil_div(b.rows, 256), 256, symmetric) >= sms) return ns_launch<256>(a, b, e, batch, symmetric);
  if (batch * (int64_t)ns_tiles((int)tm, (int)ceil_div(b.rows, 128), 128, symmetric) * 2 >= sms) return ns_launch<128>(a, b, e, batch, symmetric);
  return ns_launch<64>(a, b, e, batch, symmetric);
}

}  // namespace b200
