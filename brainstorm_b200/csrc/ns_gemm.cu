// out = alpha a b^T + diagonal I in fp32 accuracy on tcgen05.mma kind::f16, for operands that are already split
// into two half-precision planes (hi = fp16(x), lo = fp16(x - hi), 22 bits together): what the Newton-Schulz
// iteration of muon.cu multiplies.  Its matrices stay below 4 in magnitude, so one fixed scale keeps them in
// the range of half precision, and the epilogue of one product writes the planes the next one reads: nothing
// is split inside the main loop.
//
//  * a b = hi.hi + hi.lo + lo.hi: three MMAs for each step of 16 along K, at twice the rate and half the operand
//    bytes of three TF32 MMAs of depth 8.
//  * Operands lie as they are: K along the rows (K-major) or across them (MN-major), both in the 128-byte swizzle, so
//    nothing is ever transposed in memory.
//  * Large products run on pairs of SMs (cta_group::2, 256 x 256 tiles), smaller ones on single SMs (128 x 128,
//    128 x 64).  Bound: shared memory, 128 bytes a clock.  Per MMA of depth 16 a single SM reads 8 KB of operands of a
//    128 x 128 tile and TMA writes 5.3 KB: 104 clocks against the 64 of the tensor pipe (measured 120).  A 128 x 256
//    tile on one SM wants 12 + 8 KB, 156 clocks against 128 (measured 165, and two stages do not cover a load); the
//    pair stages half of b on each side.
//  * The tensor core truncates when it adds into its accumulator.  Every 64 along K (128 on pairs) are therefore a
//    chunk of their own, in each k-block the small products first; the finished chunk is added to fp32 registers
//    with rounding while the next runs in the other half of tensor memory.  On pairs the way of a chunk from the
//    issuing SM to the drain warps of both and back is longer than the MMAs of 64 along K: with such chunks a
//    4096 x 4096 update took a quarter longer than with 128.
//  * Roles (320 threads): warp 0 TMA, warp 1 MMA and tensor memory, warps 2 to 9 drain and epilogue (a lane owns
//    a row; two groups of four warps own half the columns each).  One thread issues the MMAs; the descriptors
//    of stages and steps are additions to one (with a descriptor built for each, issue took 180 clocks an MMA), and the
//    thread is elected, not picked by lane == 0, so that they stay in uniform registers (twelve MMAs: 500 to 660 clocks
//    to issue instead of 1000 to 1380; a 4096 x 4096 update 4.21 -> 3.88 ms).
//  * A symmetric product computes and stores the blocks on and above the diagonal.  Where a product needs a block
//    below it, the block above is loaded as an MN-major operand in its place: K-block by K-block, the
//    instruction descriptor says which.  (Storing both halves made the epilogue cost 0.15 ms of a 0.51 ms update of four
//    1000 x 1000 matrices.)
//  * Every wait is bounded, as in the general GEMM.
#include <cuda.h>

#include <algorithm>

#include "half_split.cuh"
#include "ns_gemm.cuh"
#include "tc_ptx.cuh"

namespace b200 {

int* device_error_flag();       // gemm_tc.cu

constexpr int NS_BM = 128, NS_THREADS = 320;

// BN: columns of a tile; PAIR: the tile is 256 x 256, this CTA holds 128 rows of a, 128 rows of b and 128 x 256 of the
// accumulator.
template <int BN_, bool PAIR>
struct NsConfig {
  static constexpr int BN = BN_, BK = 64, B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int A_BYTES = NS_BM * BK * 2, B_BYTES = B_ROWS * BK * 2;        // one plane
  static constexpr int STAGE_BYTES = 2 * (A_BYTES + B_BYTES);
  static constexpr int STAGES = 196608 / STAGE_BYTES;
  static constexpr int CHUNK = (PAIR ? 128 : 64) / BK;                             // stages between two drains
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int ACC = BN / 2;                                               // columns of a drain group
  static constexpr int W = BN == 128 ? 64 : 32;                                    // columns of an epilogue step
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
  // Descriptors, both in the 128-byte swizzle.  K-major: rows of 64 halves, eight of them one group.  MN-major: boxes of 64
  // K-rows x 64 operand rows (128 bytes a K-row), eight K-rows one group.
  __device__ static uint64_t desc_k(uint32_t at) { return smem_desc(at, 16, 1024, 2); }
  __device__ static uint64_t desc_mn(uint32_t at) { return smem_desc(at, BK * 128, 1024, 2); }
};
using NsPair = NsConfig<256, true>;
using Ns128 = NsConfig<128, false>;
using Ns64 = NsConfig<64, false>;

struct NsOut {
  __half* data;
  int ld;
  float alpha, diagonal;
};
// How an operand lies: 0 K-major, 1 MN-major, else symmetric with blocks of that many rows (NsMatrix::upper).
__device__ __forceinline__ bool ns_mn(int lies, int r0, int k0) { return lies <= 1 ? lies : k0 / lies < r0 / lies; }

// Tile t of the walk: bands of 8 row tiles, column by column inside a band, so that the blocks that run
// together share rows of both operands in L2.  Symmetric: only tiles that reach the diagonal or lie above it.
__device__ __forceinline__ bool ns_tile(int t, int tiles_m, int tiles_n, int bm, int bn, bool symmetric, int* i, int* j) {
  for (int band = 0; band < tiles_m; band += 8) {
    const int rows = min(8, tiles_m - band);
    for (int c = symmetric ? band * bm / bn : 0; c < tiles_n; ++c) {
      // rows of this band whose tile at column c reaches the diagonal: bm i <= bn (c + 1) - 1
      const int fit = symmetric ? min(rows, (bn * (c + 1) - 1) / bm - band + 1) : rows;
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
static int ns_tiles(int tiles_m, int tiles_n, int bm, int bn, bool symmetric) {
  if (!symmetric) return tiles_m * tiles_n;
  int n = 0;
  for (int band = 0; band < tiles_m; band += 8) {
    const int rows = std::min(8, tiles_m - band);
    for (int c = band * bm / bn; c < tiles_n; ++c) n += std::min(rows, (bn * (c + 1) - 1) / bm - band + 1);
  }
  return n;
}

// W columns (64 or 32) of a warp's 32 rows: from acc (lane: row row0 + lane; columns col ..) to the planes.  Rows go
// through shared memory (`buf`, this warp's: both planes, 32 rows of W halves and 16 bytes), so that whole rows of a
// tile meet global memory together: a lane that stored its own row touched 32 lines an instruction, which made the
// epilogue of a 128 x 256 tile take 33 to 56 thousand clocks beside a main loop of 133 thousand (K = 4096).
template <int W>
__device__ __forceinline__ void ns_store(const float* acc, uint8_t* buf, const NsOut& e, int64_t plane, int row0, int col, int M) {
  constexpr int PITCH = W * 2 + 16, PLANE = 32 * PITCH, LPR = W / 8, RPI = 32 / LPR;     // lanes per row, rows per instruction
  const int lane = threadIdx.x & 31;
  uint8_t* mine = buf + lane * PITCH;
  const float alpha = e.alpha / NS_SCALE, diagonal = e.diagonal * NS_SCALE;
  const int on = row0 + lane - col;                        // the diagonal's place among this lane's columns
#pragma unroll
  for (int c8 = 0; c8 < W / 8; ++c8) {
    uint32_t hi[4], lo[4];
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = alpha * acc[8 * c8 + u] + (on == 8 * c8 + u ? diagonal : 0.f);
#pragma unroll
    for (int u = 0; u < 4; ++u) split_halves(x[2 * u], x[2 * u + 1], hi[u], lo[u]);
    *reinterpret_cast<uint4*>(mine + 16 * c8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(mine + PLANE + 16 * c8) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  __syncwarp();
  const int lr = lane / LPR, lc = col + 8 * (lane % LPR);
#pragma unroll
  for (int i = 0; i < LPR; ++i) {
    const int r = row0 + lr + RPI * i;
    const uint8_t* from = buf + (lr + RPI * i) * PITCH + 16 * (lane % LPR);
    const uint4 h = *reinterpret_cast<const uint4*>(from), l = *reinterpret_cast<const uint4*>(from + PLANE);
    if (r >= M || lc >= e.ld) continue;
    __half* at = e.data + (int64_t)r * e.ld + lc;
    *reinterpret_cast<uint4*>(at) = h;
    *reinterpret_cast<uint4*>(at + plane) = l;
  }
  __syncwarp();
}

// The end of a drain warp's work: its 32 rows x ACC columns.
template <class Cfg>
__device__ __forceinline__ void ns_finish(const float (&acc)[Cfg::ACC], uint8_t* smem, int drain_warp, NsOut e, int row0, int col0, int M, int N,
                                          int b, int batch) {
  constexpr int W = Cfg::W;
  static_assert(8 * 2 * 32 * (W * 2 + 16) <= Cfg::STAGES * Cfg::STAGE_BYTES, "epilogue staging does not fit");
  uint8_t* buf = smem + drain_warp * 2 * 32 * (W * 2 + 16);
  e.data += (int64_t)b * M * e.ld;
  const int64_t plane = (int64_t)batch * M * e.ld;
  if (row0 >= M) return;
#pragma unroll
  for (int cc = 0; cc < Cfg::ACC / W; ++cc)
    if (col0 + W * cc < N) ns_store<W>(acc + W * cc, buf, e, plane, row0, col0 + W * cc, M);
}

// ROWS rows of an operand from r0, BK along K from k0, both planes, into the stage at `at`.
template <int ROWS, int BK>
__device__ __forceinline__ void ns_load(uint32_t at, const CUtensorMap* map, const CUtensorMap* map_mn, bool mn, int k0, int r0, int batch, int b,
                                        uint32_t bar) {
#pragma unroll
  for (int plane = 0; plane < 2; ++plane) {
    const uint32_t to = at + plane * ROWS * BK * 2;
    if (!mn) {
      tma_load_3d(to, map, k0, r0, plane * batch + b, bar);
    } else {
#pragma unroll
      for (int j = 0; j < ROWS / 64; ++j) tma_load_3d(to + j * BK * 128, map_mn, r0 + 64 * j, k0, plane * batch + b, bar);
    }
  }
}

template <class Cfg>
__global__ void __launch_bounds__(NS_THREADS, 1)
ns_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a_mn, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_b_mn, NsOut e, int M, int N, int K, int batch,
               int a_lies, int b_lies, int symmetric, int* error_flag) {
  constexpr int S = Cfg::STAGES, BN = Cfg::BN, BK = Cfg::BK, CH = Cfg::CHUNK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * Cfg::STAGE_BYTES);
  // bars[0..S) full, [S..2S) empty, [2S..2S+2) chunk ready, [2S+2..2S+4) chunk drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  int ti = 0, tj = 0;
  ns_tile(blockIdx.x, (M + NS_BM - 1) / NS_BM, (N + BN - 1) / BN, NS_BM, BN, symmetric, &ti, &tj);
  const int m0 = ti * NS_BM, n0 = tj * BN;
  const int num_kb = (K + BK - 1) / BK;
  const uint32_t bar0 = smem_u32(bars), smem_base = smem_u32(smem);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto acc_full_bar = [&](int i) { return bar0 + 8u * (2 * S + i); };
  auto acc_empty_bar = [&](int i) { return bar0 + 8u * (2 * S + 2 + i); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full_bar(i), 1);
      mbar_init(acc_empty_bar(i), 8);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_launch_dependents();
  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a_mn) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b_mn) : "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_d = *tmem_slot;
  pdl_wait();       // operands and outputs belong to the kernel before until here

  if (warp == 0) {
    if (elect_one()) {
      asm volatile("fence.proxy.async;" ::: "memory");      // the planes were written by ordinary stores
      int issued = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        const int s = kb % S;
        if (!mbar_wait(empty_bar(s), ((kb / S) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(full_bar(s), Cfg::STAGE_BYTES);
        const uint32_t at = smem_base + s * Cfg::STAGE_BYTES;
        ns_load<NS_BM, BK>(at, &map_a, &map_a_mn, ns_mn(a_lies, m0, kb * BK), kb * BK, m0, batch, b, full_bar(s));
        ns_load<BN, BK>(at + 2 * Cfg::A_BYTES, &map_b, &map_b_mn, ns_mn(b_lies, n0, kb * BK), kb * BK, n0, batch, b, full_bar(s));
        issued = kb + 1;
      }
      if (*abort_flag) {        // copies already issued must land before shared memory is released
        for (int kb = issued > S ? issued - S : 0; kb < issued; ++kb)
          for (uint32_t it = 0; it < TC_SPIN_LIMIT && !mbar_try_wait(full_bar(kb % S), (kb / S) & 1); ++it) __nanosleep(64);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      // D = F32, A = B = F16, N >> 3, M >> 4; the majors are set for each k-block
      const uint32_t idesc0 = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(NS_BM >> 4) << 24);
      // descriptors of stage 0; stages, planes and steps along K are additions to their address field (16-byte units)
      const uint64_t da_k = Cfg::desc_k(smem_base), da_mn = Cfg::desc_mn(smem_base);
      const uint64_t db_k = Cfg::desc_k(smem_base + 2 * Cfg::A_BYTES), db_mn = Cfg::desc_mn(smem_base + 2 * Cfg::A_BYTES);
      bool ok = true;
      int s = 0;
      for (int kb = 0; kb < num_kb; ++kb, s = s + 1 == S ? 0 : s + 1) {
        const int chunk = kb / CH, buf = chunk & 1;
        const bool fresh = kb % CH == 0, last = kb % CH == CH - 1 || kb == num_kb - 1;
        if (fresh) ok = mbar_wait(acc_empty_bar(buf), ((chunk >> 1) & 1) ^ 1, abort_flag);
        ok = ok && mbar_wait(full_bar(s), (kb / S) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const bool a_mn = ns_mn(a_lies, m0, kb * BK), b_mn = ns_mn(b_lies, n0, kb * BK);
        const uint32_t idesc = idesc0 | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
        const uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;       // 16 K-rows of 128 bytes, or 32 bytes
        const uint32_t d = tmem_d + (uint32_t)(buf * BN);
        const uint64_t ah = (a_mn ? da_mn : da_k) + (uint64_t)(s * (Cfg::STAGE_BYTES >> 4)), al = ah + (Cfg::A_BYTES >> 4);
        const uint64_t bh = (b_mn ? db_mn : db_k) + (uint64_t)(s * (Cfg::STAGE_BYTES >> 4)), bl = bh + (Cfg::B_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {          // the small products first
          mma_f16(d, al + a_step * k, bh + b_step * k, idesc, !(fresh && k == 0));
          mma_f16(d, ah + a_step * k, bl + b_step * k, idesc, 1);
        }
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) mma_f16(d, ah + a_step * k, bh + b_step * k, idesc, 1);
        mma_commit(empty_bar(s));
        if (last) mma_commit(acc_full_bar(buf));
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, group = (warp - 2) >> 2;    // tensor-memory lanes, columns of this warp
    const uint32_t lane_bits = (uint32_t)(q * 32) << 16;
    float acc[Cfg::ACC];
#pragma unroll
    for (int j = 0; j < Cfg::ACC; ++j) acc[j] = 0.f;
    bool ok = true;
    const int chunks = (num_kb + CH - 1) / CH;
    for (int chunk = 0; chunk < chunks && ok; ++chunk) {
      const int buf = chunk & 1;
      ok = mbar_wait(acc_full_bar(buf), (chunk >> 1) & 1, abort_flag);
      __syncwarp();
      if (!ok) break;
      tc_fence_after();
      drain_add<Cfg::ACC>(tmem_d + lane_bits + (uint32_t)(buf * BN + group * Cfg::ACC), acc);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty_bar(buf));
    }
    // every MMA has completed (the last chunk is drained): the stages are free
    if (__all_sync(0xffffffffu, ok)) ns_finish<Cfg>(acc, smem, warp - 2, e, m0 + q * 32, n0 + group * Cfg::ACC, M, N, b, batch);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_d, Cfg::TMEM_COLS);
  }
  if (threadIdx.x == 0 && *abort_flag && error_flag) *error_flag = 1;
}

// The same on pairs of SMs: two CTAs of a cluster (consecutive blockIdx.x) compute a 256 x 256 tile.  Each stages its own
// 128 rows of a and its own 128 of the 256 rows of b; one thread of rank 0 issues the MMAs, which read both CTAs'
// stages and leave each CTA's 128 x 256 of the product in its own tensor memory.  Rank 1's warp 1 tells rank 0
// when its tiles have landed; "stage free" and "chunk ready" are committed to both.  Set-up and the release of
// tensor memory stand between cluster barriers.
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NS_THREADS, 1)
ns_gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a_mn, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CUtensorMap map_b_mn, NsOut e, int M, int N, int K, int batch,
                    int a_lies, int b_lies, int symmetric, int* error_flag) {
  using Cfg = NsPair;
  constexpr int S = Cfg::STAGES, BN = Cfg::BN, BK = Cfg::BK, CH = Cfg::CHUNK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * Cfg::STAGE_BYTES);
  // bars[0..S) full, [S..2S) empty, [2S..3S) the peer's tiles landed (rank 0's count), then chunk ready x 2, chunk drained x 2
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const uint32_t rank = cluster_rank();
  int ti = 0, tj = 0;
  ns_tile(blockIdx.x >> 1, (M + 255) / 256, (N + 255) / 256, 256, 256, symmetric, &ti, &tj);
  const int m0 = ti * 256 + 128 * (int)rank, n0 = tj * 256;
  // One instruction descriptor serves both CTAs.  With blocks of 128 the K-blocks of the tile's own first 128 are taken
  // across the rows for both: they lie on the diagonal for the one and are stored above it for the other.
  const int a_r = ti * 256 + (a_lies == 128 ? 128 : 0), b_r = n0 + (b_lies == 128 ? 128 : 0);
  const int num_kb = (K + BK - 1) / BK;
  const uint32_t bar0 = smem_u32(bars), smem_base = smem_u32(smem);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto peer_bar = [&](int s) { return bar0 + 8u * (2 * S + s); };
  auto acc_full_bar = [&](int i) { return bar0 + 8u * (3 * S + i); };
  auto acc_empty_bar = [&](int i) { return bar0 + 8u * (3 * S + 2 + i); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
      mbar_init(peer_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full_bar(i), 1);
      mbar_init(acc_empty_bar(i), 16);       // the drain warps of both CTAs
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_launch_dependents();
  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a_mn) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b_mn) : "memory");
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_d = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      asm volatile("fence.proxy.async;" ::: "memory");
      int issued = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        const int s = kb % S;
        if (!mbar_wait(empty_bar(s), ((kb / S) & 1) ^ 1, abort_flag)) break;
        mbar_expect_tx(full_bar(s), Cfg::STAGE_BYTES);
        const uint32_t at = smem_base + s * Cfg::STAGE_BYTES;
        ns_load<NS_BM, BK>(at, &map_a, &map_a_mn, ns_mn(a_lies, a_r, kb * BK), kb * BK, m0, batch, b, full_bar(s));
        ns_load<128, BK>(at + 2 * Cfg::A_BYTES, &map_b, &map_b_mn, ns_mn(b_lies, b_r, kb * BK), kb * BK, n0 + 128 * (int)rank, batch, b, full_bar(s));
        issued = kb + 1;
      }
      if (*abort_flag) {
        for (int kb = issued > S ? issued - S : 0; kb < issued; ++kb)
          for (uint32_t it = 0; it < TC_SPIN_LIMIT && !mbar_try_wait(full_bar(kb % S), (kb / S) & 1); ++it) __nanosleep(64);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool one = elect_one();
    if (one && rank == 1) {
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(full_bar(kb % S), (kb / S) & 1, abort_flag)) break;
        mbar_arrive_cluster(cluster_addr(peer_bar(kb % S), 0));
      }
    } else if (one) {
      // D = F32, A = B = F16, N >> 3, M >> 4; the majors are set for each k-block
      const uint32_t idesc0 = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
      // descriptors of stage 0; stages, planes and steps along K are additions to their address field (16-byte units)
      const uint64_t da_k = Cfg::desc_k(smem_base), da_mn = Cfg::desc_mn(smem_base);
      const uint64_t db_k = Cfg::desc_k(smem_base + 2 * Cfg::A_BYTES), db_mn = Cfg::desc_mn(smem_base + 2 * Cfg::A_BYTES);
      bool ok = true;
      int s = 0;
      for (int kb = 0; kb < num_kb; ++kb, s = s + 1 == S ? 0 : s + 1) {
        const int chunk = kb / CH, buf = chunk & 1;
        const bool fresh = kb % CH == 0, last = kb % CH == CH - 1 || kb == num_kb - 1;
        if (fresh) ok = mbar_wait_cluster(acc_empty_bar(buf), ((chunk >> 1) & 1) ^ 1, abort_flag);
        ok = ok && mbar_wait(full_bar(s), (kb / S) & 1, abort_flag) && mbar_wait_cluster(peer_bar(s), (kb / S) & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const bool a_mn = ns_mn(a_lies, a_r, kb * BK), b_mn = ns_mn(b_lies, b_r, kb * BK);
        const uint32_t idesc = idesc0 | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
        const uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;       // 16 K-rows of 128 bytes, or 32 bytes
        const uint32_t d = tmem_d + (uint32_t)(buf * BN);
        const uint64_t ah = (a_mn ? da_mn : da_k) + (uint64_t)(s * (Cfg::STAGE_BYTES >> 4)), al = ah + (Cfg::A_BYTES >> 4);
        const uint64_t bh = (b_mn ? db_mn : db_k) + (uint64_t)(s * (Cfg::STAGE_BYTES >> 4)), bl = bh + (Cfg::B_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          mma_f16_pair(d, al + a_step * k, bh + b_step * k, idesc, !(fresh && k == 0));
          mma_f16_pair(d, ah + a_step * k, bl + b_step * k, idesc, 1);
        }
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) mma_f16_pair(d, ah + a_step * k, bh + b_step * k, idesc, 1);
        mma_commit_pair(empty_bar(s));                       // this CTA's stage and chunk, and the peer's
        mma_commit_pair(cluster_addr(empty_bar(s), 1));
        if (last) {
          mma_commit_pair(acc_full_bar(buf));
          mma_commit_pair(cluster_addr(acc_full_bar(buf), 1));
        }
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, group = (warp - 2) >> 2;
    const uint32_t lane_bits = (uint32_t)(q * 32) << 16;
    float acc[Cfg::ACC];
#pragma unroll
    for (int j = 0; j < Cfg::ACC; ++j) acc[j] = 0.f;
    bool ok = true;
    const int chunks = (num_kb + CH - 1) / CH;
    for (int chunk = 0; chunk < chunks && ok; ++chunk) {
      const int buf = chunk & 1;
      ok = mbar_wait(acc_full_bar(buf), (chunk >> 1) & 1, abort_flag);
      __syncwarp();
      if (!ok) break;
      tc_fence_after();
      drain_add<Cfg::ACC>(tmem_d + lane_bits + (uint32_t)(buf * BN + group * Cfg::ACC), acc);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(acc_empty_bar(buf), 0));
    }
    if (__all_sync(0xffffffffu, ok)) ns_finish<Cfg>(acc, smem, warp - 2, e, m0 + q * 32, n0 + group * Cfg::ACC, M, N, b, batch);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();        // nobody in the pair reads shared or tensor memory of the other any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_d, Cfg::TMEM_COLS);
  }
  if (threadIdx.x == 0 && *abort_flag && error_flag) *error_flag = 1;
}

typedef CUresult (*NsEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Both planes of a stack: along the rows, rows, then plane and matrix.  K-major boxes of 64 x rows, MN-major 64 x 64.
static int ns_map(const NsMatrix& a, bool mn, int batch, int rows, CUtensorMap* out) {
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
  const cuuint32_t box[3] = {64u, mn ? 64u : (cuuint32_t)rows, 1u}, one[3] = {1u, 1u, 1u};
  const CUresult r = encode(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return B200_OK;
}

// What the truncating accumulation of a chunk takes from a sum of one sign, on the average: without it one Newton-Schulz step
// makes X too small by 2 to 9e-7 at every shape tried.  Chosen at seven shapes from 64 x 3000 to 4096 x 4096; at others, in all forms of the
// products, the error against 64 bits of one step / of five, without it and with it:
//   16 x 65     3.4e-7 / 1.4e-6   1.7e-7 / 1.6e-6        300 x 700              4.5e-7 / 2.0e-6   2.1e-7 / 0.8e-6
//   64 x 65     6.4e-7 / 4.0e-6   3.1e-7 / 2.0e-6        513 x 640              4.8e-7 / 2.2e-6   2.0e-7 / 0.9e-6
//   130 x 129   6.0e-7 / 3.9e-6   2.8e-7 / 1.9e-6        30 x 210 x 215         5.7e-7 / 2.0e-6   2.7e-7 / 0.9e-6
//   128 x 193   5.9e-7 / 3.6e-6   2.8e-7 / 1.6e-6        40 x 165 x 170         7.4e-7 / 3.6e-6   4.1e-7 / 1.9e-6
//   48 x 200    5.6e-7 / 3.1e-6   2.5e-7 / 1.1e-6        20 x 390 x 395         9.4e-7 / 4.4e-6   6.2e-7 / 2.9e-6
//   20 x 20     4.9e-7 / 2.0e-6   2.2e-7 / 1.0e-6        2100 x 2100            3.1e-7 / 3.4e-6   2.6e-7 / 1.9e-6
// A sum of up to 8 products truncates little; there the factor is an error of its own size: 1 x 1 0.9e-7 / 6.1e-7 and 2.6e-7 / 0.8e-7,
// 3 x 7 2.1e-7 / 2.1e-7 and 2.7e-7 / 7.4e-7, 4 x 4 2.1e-7 / 5.0e-7 and 2.1e-7 / 7.0e-7, 8 x 8 2.4e-7 / 1.2e-6 and 2.3e-7 / 1.3e-6.
constexpr float NS_GAIN = 1.f + 0x1p-22f;

typedef void (*NsKernel)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap, NsOut, int, int, int, int, int, int, int, int*);

int ns_gemm(const NsMatrix& a, bool a_t, const NsMatrix& b, bool b_t, NsMatrix* out, int batch, float alpha, float diagonal, bool symmetric) {
  // tile height and width, SMs of a tile, clocks for 64 along K (12 MMAs; measured), rows of b in a box
  struct Form {
    NsKernel kernel;
    int bm, bn, sms, clocks, b_rows, smem;
  };
  static const Form forms[] = {{(NsKernel)ns_gemm_kernel<Ns128>, 128, 128, 1, 1450, 128, Ns128::SMEM_BYTES},
                               {(NsKernel)ns_gemm_kernel<Ns64>, 128, 64, 1, 1320, 64, Ns64::SMEM_BYTES},
                               {(NsKernel)ns_gemm_pair_kernel, 256, 256, 2, 1700, 128, NsPair::SMEM_BYTES}};
  static bool ready = false;
  if (!ready) {
    for (const Form& f : forms) B200_CUDA(cudaFuncSetAttribute(f.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, f.smem));
    ready = true;
  }
  int* flag = device_error_flag();
  B200_REQUIRE(flag != nullptr, "the device error flag cannot be set up");
  const int M = out->rows, N = out->cols, K = a_t ? a.rows : a.cols;
  const NsOut e = {out->data, out->ld, alpha * NS_GAIN, diagonal};
  // the form with the least waves times clocks
  const Form* best = nullptr;
  int64_t least = 0;
  int tiles = 0;
  for (const Form& f : forms) {
    const int t = ns_tiles((int)ceil_div(M, f.bm), (int)ceil_div(N, f.bn), f.bm, f.bn, symmetric);
    const int64_t cost = ceil_div((int64_t)t * batch, state().sm_count / f.sms) * f.clocks;
    if (!best || cost < least) {
      best = &f;
      least = cost;
      tiles = t * f.sms;
    }
  }
  out->upper = symmetric ? std::max(best->bm, best->bn) < 256 ? 128 : 256 : 0;
  CUtensorMap ma, ma_mn, mb, mb_mn;
  if (int rc = ns_map(a, false, batch, NS_BM, &ma)) return rc;
  if (int rc = ns_map(a, true, batch, NS_BM, &ma_mn)) return rc;
  if (int rc = ns_map(b, false, batch, best->b_rows, &mb)) return rc;
  if (int rc = ns_map(b, true, batch, best->b_rows, &mb_mn)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)tiles, (unsigned)batch);
  cfg.blockDim = dim3(NS_THREADS);
  cfg.dynamicSmemBytes = best->smem;
  cfg.stream = state().stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  B200_CUDA(cudaLaunchKernelEx(&cfg, best->kernel, ma, ma_mn, mb, mb_mn, e, M, N, K, batch, a.upper ? a.upper : (int)a_t, b.upper ? b.upper : (int)b_t,
                               symmetric ? 1 : 0, flag));
  B200_LAUNCH_CHECK();
  return B200_OK;
}

// ---- the whole iteration in one launch, for matrices of a few tiles
//
// A product of such matrices is all latency: launched one by one, those of 205 x 256 take 6.2 us each (an update 107.7 us,
// 96.3 in a recorded graph), of which the tensor pipe has work for one.  Here a cluster of up to eight CTAs computes all
// of them for one matrix of the stack: the operands stay in L2, barriers and tensor memory are set up once, and between two
// products stands a barrier of the cluster (with a fence between the stores of the one and the TMA loads of the next)
// instead of a launch: 92 us, 89 recorded; 64 x 64: 65.8 -> 57.5, eight of 128 x 256: 95.4 -> 81.6.  Of a product's
// 9000 clocks then 1500 are the way to the first MMA, 4000 the four K-blocks (loads and MMAs share the 128 bytes a clock
// of shared memory), 2000 the epilogue, 1500 fence and barrier.
// With two tiles a CTA it lost (256 x 500: 122.6 recorded against 116.0), as with more clusters than fit the GPU together
// (sixteen of 256 x 256: 178 against 116): each CTA has one tile, and there are at most 64 tiles.
constexpr int NC_CTAS = 8;

struct NsChain {
  __half* data[4];                                   // X, the other X, D, P
  int ld[4];
  int rows, cols, m, steps, tall, batch;
  float d_diagonal, p_alpha, p_diagonal;
};
// ROWS rows of an operand as ns_load, with one map for both majors: the boxes are 64 x 64 either way.
template <int ROWS>
__device__ __forceinline__ void ns_chain_load(uint32_t at, const CUtensorMap* map, bool mn, int k0, int r0, int batch, int b, uint32_t bar) {
#pragma unroll
  for (int plane = 0; plane < 2; ++plane)
#pragma unroll
    for (int j = 0; j < ROWS / 64; ++j)
      tma_load_3d(at + plane * ROWS * 128 + j * 8192, map, mn ? r0 + 64 * j : k0, mn ? k0 : r0 + 64 * j, plane * batch + b, bar);
}

struct NcConfig : NsConfig<64, false> {
  static constexpr int STAGES = 3, OUT_BYTES = 8 * 2 * 32 * (W * 2 + 16);
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + OUT_BYTES + 1024 + 256;
};

__global__ void __launch_bounds__(NS_THREADS, 1)
ns_chain_kernel(const __grid_constant__ CUtensorMap map0, const __grid_constant__ CUtensorMap map1, const __grid_constant__ CUtensorMap map2,
                const __grid_constant__ CUtensorMap map3, const __grid_constant__ NsChain c, int* error_flag) {
  using Cfg = NcConfig;
  constexpr int S = Cfg::STAGES, BN = Cfg::BN, BK = Cfg::BK;
  static_assert(Cfg::CHUNK == 1 && BK == 64, "a stage is a chunk");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S * Cfg::STAGE_BYTES + Cfg::OUT_BYTES);
  // bars[0..S) full, [S..2S) empty, [2S..2S+2) chunk ready, [2S+2..2S+4) chunk drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y, rank = blockIdx.x;       // a cluster is a row of the grid
  const uint32_t bar0 = smem_u32(bars), smem_base = smem_u32(smem);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto acc_full_bar = [&](int i) { return bar0 + 8u * (2 * S + i); };
  auto acc_empty_bar = [&](int i) { return bar0 + 8u * (2 * S + 2 + i); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full_bar(i), 1);
      mbar_init(acc_empty_bar(i), 8);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map0) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map1) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map2) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map3) : "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_d = *tmem_slot;

  // Every role counts its stages (a stage is a chunk) through all products.
  int s = 0, phase = 0, buf = 0, buf_phase = 0;
  uint32_t issued = 0;
  bool ok = true;
  auto advance = [&]() {
    if (++s == S) s = 0, phase ^= 1;
    buf ^= 1;
    if (buf == 0) buf_phase ^= 1;
  };
  // this CTA's tile of D and P, and of X: row tile << 16 | column tile, -1 for none
  int mine[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int M = w == 0 ? c.m : c.rows, N = w == 0 ? c.m : c.cols;
    int ti = 0, tj = 0;
    const bool any = ns_tile(rank, (M + NS_BM - 1) / NS_BM, (N + BN - 1) / BN, NS_BM, BN, w == 0, &ti, &tj);
    mine[w] = any ? ti << 16 | tj : -1;
  }
  pdl_wait();
  for (int x = 0, step = 0; step < c.steps; ++step, x ^= 1) {
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      // D = X X^T (X^T X) + .. I, P = c D D + .. I, X' = P X (X P)
      const CUtensorMap* map_x = x ? &map1 : &map0;
      const CUtensorMap* map_a = w == 0 ? map_x : w == 1 ? &map2 : c.tall ? map_x : &map3;
      const CUtensorMap* map_b = w == 0 ? map_x : w == 1 ? &map2 : c.tall ? &map3 : map_x;
      const int a_lies = w == 0 ? c.tall : w == 1 || !c.tall ? 128 : 0, b_lies = w == 0 ? c.tall : w == 1 || c.tall ? 128 : 1;
      const int M = w < 2 ? c.m : c.rows, N = w < 2 ? c.m : c.cols, K = w > 0 ? c.m : c.tall ? c.rows : c.cols;
      const int num_kb = (K + BK - 1) / BK;
      const int t = mine[w == 2];
      if (t >= 0 && ok) {
        const int m0 = (t >> 16) * NS_BM, n0 = (t & 0xffff) * BN;
        if (warp == 0) {
          if (elect_one()) {
            asm volatile("fence.proxy.async;" ::: "memory");      // the operands were written by ordinary stores
            for (int kb = 0; kb < num_kb; ++kb) {
              ok = mbar_wait(empty_bar(s), phase ^ 1, abort_flag);
              if (!ok) break;
              mbar_expect_tx(full_bar(s), Cfg::STAGE_BYTES);
              const uint32_t at = smem_base + s * Cfg::STAGE_BYTES;
              ns_chain_load<NS_BM>(at, map_a, ns_mn(a_lies, m0, kb * BK), kb * BK, m0, c.batch, b, full_bar(s));
              ns_chain_load<BN>(at + 2 * Cfg::A_BYTES, map_b, ns_mn(b_lies, n0, kb * BK), kb * BK, n0, c.batch, b, full_bar(s));
              ++issued;
              advance();
            }
          }
        } else if (warp == 1) {
          if (elect_one()) {
            const uint32_t idesc0 = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(NS_BM >> 4) << 24);
            const uint64_t da_k = Cfg::desc_k(smem_base), da_mn = Cfg::desc_mn(smem_base);
            const uint64_t db_k = Cfg::desc_k(smem_base + 2 * Cfg::A_BYTES), db_mn = Cfg::desc_mn(smem_base + 2 * Cfg::A_BYTES);
            for (int kb = 0; kb < num_kb; ++kb) {
              ok = mbar_wait(acc_empty_bar(buf), buf_phase ^ 1, abort_flag) && mbar_wait(full_bar(s), phase, abort_flag);
              if (!ok) break;
              tc_fence_after();
              const bool a_mn = ns_mn(a_lies, m0, kb * BK), b_mn = ns_mn(b_lies, n0, kb * BK);
              const uint32_t idesc = idesc0 | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16);
              const uint32_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
              const uint32_t d = tmem_d + (uint32_t)(buf * BN);
              const uint64_t ah = (a_mn ? da_mn : da_k) + (uint64_t)(s * (Cfg::STAGE_BYTES >> 4)), al = ah + (Cfg::A_BYTES >> 4);
              const uint64_t bh = (b_mn ? db_mn : db_k) + (uint64_t)(s * (Cfg::STAGE_BYTES >> 4)), bl = bh + (Cfg::B_BYTES >> 4);
#pragma unroll
              for (int k = 0; k < BK / 16; ++k) {
                mma_f16(d, al + a_step * k, bh + b_step * k, idesc, k > 0);
                mma_f16(d, ah + a_step * k, bl + b_step * k, idesc, 1);
              }
#pragma unroll
              for (int k = 0; k < BK / 16; ++k) mma_f16(d, ah + a_step * k, bh + b_step * k, idesc, 1);
              mma_commit(empty_bar(s));
              mma_commit(acc_full_bar(buf));
              advance();
            }
          }
        } else {
          const int q = warp & 3, group = (warp - 2) >> 2;
          float acc[Cfg::ACC];
#pragma unroll
          for (int j = 0; j < Cfg::ACC; ++j) acc[j] = 0.f;
          for (int kb = 0; kb < num_kb; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full_bar(buf), buf_phase, abort_flag));
            if (!ok) break;
            tc_fence_after();
            drain_add<Cfg::ACC>(tmem_d + ((uint32_t)(q * 32) << 16) + (uint32_t)(buf * BN + group * Cfg::ACC), acc);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty_bar(buf));
            advance();
          }
          const int row0 = m0 + q * 32, col0 = n0 + group * Cfg::ACC;
          if (ok && row0 < M && col0 < N) {
            const int out = w < 2 ? 2 + w : x ^ 1, ld = c.ld[out];
            const NsOut e = {c.data[out] + (int64_t)b * M * ld, ld, (w == 1 ? c.p_alpha : 1.f) * NS_GAIN, w == 0 ? c.d_diagonal : w == 1 ? c.p_diagonal : 0.f};
            ns_store<Cfg::W>(acc, smem + S * Cfg::STAGE_BYTES + (warp - 2) * 2 * 32 * (Cfg::W * 2 + 16), e, (int64_t)c.batch * M * ld, row0, col0, M);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      // the product is complete before anyone loads it: stores, fence, barrier, TMA
      __syncwarp();
      if (warp >= 2) asm volatile("fence.proxy.async;" ::: "memory");
      cluster_sync_all();
    }
  }
  if (warp == 0 && issued && *abort_flag) {      // copies already issued must land before shared memory is released
    for (uint32_t k = issued > S ? issued - S : 0; k < issued; ++k)
      for (uint32_t n = 0; n < TC_SPIN_LIMIT && !mbar_try_wait(full_bar(k % S), (k / S) & 1); ++n) __nanosleep(64);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_d, Cfg::TMEM_COLS);
  }
  if (threadIdx.x == 0 && *abort_flag && error_flag) *error_flag = 1;
}

static int ns_chain_tiles(int64_t rows, int64_t cols) { return (int)(ceil_div(rows, NS_BM) * ceil_div(cols, 64)); }

bool ns_chain_fits(int64_t rows, int64_t cols, int64_t batch) {
  return rows <= 4096 && cols <= 4096 && ns_chain_tiles(rows, cols) <= NC_CTAS && batch * ns_chain_tiles(rows, cols) <= 64;
}

int ns_chain(const NsMatrix* X, const NsMatrix& D, const NsMatrix& P, bool tall, int batch, int steps, float d_diagonal, float p_alpha, float p_diagonal) {
  static bool ready = false;
  if (!ready) {
    B200_CUDA(cudaFuncSetAttribute(ns_chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NcConfig::SMEM_BYTES));
    ready = true;
  }
  int* flag = device_error_flag();
  B200_REQUIRE(flag != nullptr, "the device error flag cannot be set up");
  int ctas = 1;
  const int full = ns_chain_tiles(X[0].rows, X[0].cols);
  while (ctas < full && ctas < NC_CTAS) ctas *= 2;
  const NsChain c = {{X[0].data, X[1].data, D.data, P.data}, {X[0].ld, X[1].ld, D.ld, P.ld}, X[0].rows, X[0].cols, D.rows, steps, tall ? 1 : 0, batch, d_diagonal, p_alpha, p_diagonal};
  CUtensorMap maps[4];
  const NsMatrix* all[4] = {&X[0], &X[1], &D, &P};
  for (int i = 0; i < 4; ++i)
    if (int rc = ns_map(*all[i], true, batch, 64, &maps[i])) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)batch);
  cfg.blockDim = dim3(NS_THREADS);
  cfg.dynamicSmemBytes = NcConfig::SMEM_BYTES;
  cfg.stream = state().stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  B200_CUDA(cudaLaunchKernelEx(&cfg, ns_chain_kernel, maps[0], maps[1], maps[2], maps[3], c, flag));
  B200_LAUNCH_CHECK();
  return B200_OK;
}

}  // namespace b200
