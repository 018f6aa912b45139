// The narrow products of the adapter operators on the tensor cores (f16 and
// bf16): the shrink Q[t, :] = s_a·P_a·X[t] and the outer sums
// dP_a = Σ_{t in a} Q[t] ⊗ X[t]. The wide product is gemm_adapted (lc_gemm.cu).
#include "lc_adapters.h"
#include "lc_api.h"
#include "lc_gemm.h"
#include "lc_sm100.cuh"

#include <algorithm>

__device__ unsigned int g_adapter_err;

namespace {
using namespace sm100;
using namespace lc;

constexpr int TC_THREADS = 192;  // TMA producer, MMA issuer, four epilogue warps
constexpr int BM = 128, BK = 64;
constexpr int SK = 128;                       // columns per stage of the shrink
constexpr uint32_t X_BYTES = BM * SK * 2;

template <typename T>
__device__ __forceinline__ uint32_t idesc_rt(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (TcFmt<T>::ab << 7) | (TcFmt<T>::ab << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
// The load is warp-wide (.aligned): the lanes meet first, since the code before
// it treats rows of a warp differently.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
// ------------------------------------------------------------- shrink
//
// One CTA takes tiles of 128 rows of one or two products (both directions of a
// gradient share a launch). Per 128 columns of X the ring holds the X block
// (TMA, 32 KB) and, for up to `nb` of the tile's segments, their blocks of P_a
// (R rows each), side by side: one MMA per 16 columns gives every row against
// every one of these adapters, D [128, n·R] (n·R <= 256), and the epilogue
// takes from each row's n results the one of its own adapter, scales, splits
// and stores it. The tensor cores have room for the others: an MMA this narrow
// costs the reading of X, not its width; one MMA per segment with the other
// rows switched off took 131 us for what takes 79. More segments than nb: the
// tile's columns are streamed again. D is double-buffered in TMEM.
//
// Bound by the read of X: 69,135 rows of 2304 and of 768 columns in f16 (424 MB),
// rank 16, take 78 us with 256 requests (5.4 TB/s, 0.83 of the measured copy);
// stages of 64 columns instead of 128 took 85. With few
// tiles the columns are split over clusters of S CTAs, whose partial D meet in
// shared memory and are added in rank order.
struct ShrinkJob {
  CUtensorMap tmX, tmP;
  __nv_bfloat16* Q;
  __half* H;
  int C, blocks;  // blocks: tmX brings both 64-column blocks of a stage (a 3-D map)
};
struct ShrinkArgs {
  ShrinkJob job[2];  // the longer one first
  int njobs, T, ntiles, R, rank, nb, stages, S;
  int extra, filled;  // the second job's tiles that even out the first's last round (ShrinkItems)
  uint32_t bank_bytes, tmem_cols;
  const int4* segs;
  const int2* tiles;
  const float* scales;
};
// The tiles of one CTA (cluster): the first job's round by round; then, where
// the last round was not full, `extra` tiles of the second job for each CTA
// that had none in it; then the rest of the second job, round by round. The
// next tile's segment range is loaded while the current tile is worked on.
struct ShrinkItems {
  const ShrinkArgs& args;
  int cta, n, rem, t, job, k = 0;
  int2 segs, ahead;  // first segment and number of segments: of this tile, of the next one
  int next_t, next_job;
  __device__ ShrinkItems(const ShrinkArgs& a, int cta_, int n_) : args(a), cta(cta_), n(n_), rem(a.ntiles % n_), next_t(cta_), next_job(0) {
    settle();
    load();
  }
  // brings (next_job, next_t) to a tile that exists, or next_job to njobs
  __device__ void settle() {
    if (next_job == 0 && next_t >= args.ntiles) {
      next_job = 1;
      next_t = -1;
    }
    if (next_job == 1 && args.njobs == 2 && next_t < 0) {
      if (cta >= rem && k < args.extra && (cta - rem) * args.extra + k < args.filled) next_t = (cta - rem) * args.extra + k++;
      else next_t = args.filled + (cta - rem + n) % n, k = args.extra;
    }
    if (next_job == 1 && (args.njobs < 2 || next_t >= args.ntiles)) next_job = 2;
  }
  __device__ void load() { ahead = next_job < args.njobs ? __ldg(args.tiles + next_t) : make_int2(0, 0); }
  __device__ bool next() {
    if (next_job >= args.njobs) return false;
    t = next_t;
    job = next_job;
    segs = ahead;
    if (next_job == 1 && k < args.extra && next_t < args.filled) next_t = -1;
    else if (next_job == 1 && next_t < args.filled) next_t = args.filled + (cta - rem + n) % n;
    else next_t += n;
    settle();
    load();
    return true;
  }
};

// Columns c .. c + N - 1 of row t of a product, into its Q and H.
template <int N>
__device__ __forceinline__ void store_q(const ShrinkJob& job, int64_t t, int R, int c, const float (&v)[N]) {
  auto put = [](auto* dst, const auto (&part)[N]) {
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 8; i++) ((uint4*)dst)[i] = ((const uint4*)part)[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) dst[i] = part[i];
    }
  };
  if (job.Q) {
    alignas(16) __nv_bfloat16 p[kQParts][N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      __nv_bfloat16 q[kQParts];
      split_bf16(v[i], q);
#pragma unroll
      for (int k = 0; k < kQParts; k++) p[k][i] = q[k];
    }
#pragma unroll
    for (int k = 0; k < kQParts; k++) put(job.Q + (t * kQParts + k) * R + c, p[k]);
  }
  if (job.H) {
    alignas(16) __half p[kHParts][N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      __half q[kHParts];
      split_f16(v[i], q);
#pragma unroll
      for (int k = 0; k < kHParts; k++) p[k][i] = q[k];
    }
#pragma unroll
    for (int k = 0; k < kHParts; k++) put(job.H + (t * kHParts + k) * R + c, p[k]);
  }
}

template <typename T>
__global__ void __launch_bounds__(TC_THREADS, 1) k_shrink_tc(const __grid_constant__ ShrinkArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t stage_bytes = X_BYTES + args.bank_bytes;
  float* sD = (float*)(smem + args.stages * stage_bytes);  // S > 1: this CTA's share of D [128, R]
  uint64_t* full = (uint64_t*)(sD + (args.S > 1 ? BM * args.R : 0));
  uint64_t* empty = full + args.stages;
  uint64_t* tfull = empty + args.stages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = (uint32_t*)(tempty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = args.S, rank = S > 1 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / S, step = gridDim.x / S;
  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], 1);
    for (int a = 0; a < 2; a++) mbar_init(&tfull[a], 1), mbar_init(&tempty[a], 4);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, args.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();  // after the wait: what runs before this kernel is done when the next one starts

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t used = 0, last_phase = 0;  // stages filled, and the phase bit of each one's last fill
      for (ShrinkItems it(args, first, step); ok && it.next();) {
        const ShrinkJob& job = args.job[it.job];
        const int KB = (job.C + SK - 1) / SK, kb0 = (int)((int64_t)rank * KB / S), kb1 = (int)((int64_t)(rank + 1) * KB / S);
        for (int s = 0; s < it.segs.y && ok; s += args.nb) {
          const int n = min(args.nb, it.segs.y - s);
          for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&empty[stage], phase ^ 1, abort, &g_adapter_err)) { ok = false; break; }
            uint8_t* st = smem + stage * stage_bytes;
            mbar_arrive_expect_tx(&full[stage], X_BYTES + (uint32_t)n * args.R * 256);
            if (job.blocks) {
              tma_load_3d(st, &job.tmX, &full[stage], 0, it.t * BM, kb * 2);
            } else {
              tma_load_2d(st, &job.tmX, &full[stage], kb * SK, it.t * BM);
              tma_load_2d(st + X_BYTES / 2, &job.tmX, &full[stage], kb * SK + 64, it.t * BM);
            }
            // (a rolled loop: unrolled over all that fit with the loads predicated, the kernel took 103 us instead of 83)
#pragma unroll 1
            for (int i = 0; i < n; i++) {
              const int a = __ldg(&args.segs[it.segs.x + s + i].z);
              tma_load_3d(st + X_BYTES + i * args.R * 128, &job.tmP, &full[stage], kb * SK, 0, a);
              tma_load_3d(st + X_BYTES + args.bank_bytes / 2 + i * args.R * 128, &job.tmP, &full[stage], kb * SK + 64, 0, a);
            }
            used |= 1u << stage;
            last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
            if (++stage == args.stages) { stage = 0; phase ^= 1; }
          }
        }
      }
      for (int s = 0; s < args.stages; s++)  // every copy issued here lands before the CTA exits
        if (used >> s & 1) {
          const uint64_t t0 = gtimer();
          while (!mbar_try_wait(&full[s], (last_phase >> s) & 1) && gtimer() - t0 < kWaitNs) {}
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      uint64_t* last = nullptr;
      uint32_t last_phase = 0;
      for (ShrinkItems it(args, first, step); ok && it.next();) {
        const ShrinkJob& job = args.job[it.job];
        const int KB = (job.C + SK - 1) / SK, kb0 = (int)((int64_t)rank * KB / S), kb1 = (int)((int64_t)(rank + 1) * KB / S);
        for (int s = 0; s < it.segs.y && ok; s += args.nb) {
          const int n = min(args.nb, it.segs.y - s);
          const uint32_t idesc = idesc_rt<T>(n * args.R, false, false);
          if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort, &g_adapter_err)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(acc * args.nb * args.R);
          for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&full[stage], phase, abort, &g_adapter_err)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a0 = smem_u32(smem + stage * stage_bytes), b0 = a0 + X_BYTES;
#pragma unroll
            for (int k = 0; k < SK / 16; k++)
              tc_mma(d, sdesc_sw128(a0 + (k / 4) * (X_BYTES / 2) + (k % 4) * 32), sdesc_sw128(b0 + (k / 4) * (args.bank_bytes / 2) + (k % 4) * 32), idesc,
                     (kb > kb0 || k > 0) ? 1u : 0u);
            tc_commit(&empty[stage]);
            last = &empty[stage];
            last_phase = phase;
            if (++stage == args.stages) { stage = 0; phase ^= 1; }
          }
          if (!ok) break;
          tc_commit(&tfull[acc]);
          last = &tfull[acc];
          last_phase = acc_phase;
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
      }
      if (last) {  // the MMAs issued here finish before TMEM is freed
        const uint64_t t0 = gtimer();
        while (!mbar_try_wait(last, last_phase) && gtimer() - t0 < kWaitNs) {}
      }
    }
  } else {
    const int quarter = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (ShrinkItems it(args, first, step); ok && it.next();) {
      const int row = it.t * BM + quarter * 32 + lane;
      for (int s = 0; s < it.segs.y && ok; s += args.nb) {
        const int n = min(args.nb, it.segs.y - s);
        if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, abort, &g_adapter_err))) { ok = false; break; }
        tc_fence_after();
        for (int i = 0; i < n; i++) {
          const int4 g = __ldg(&args.segs[it.segs.x + s + i]);
          const bool mine = row >= g.x && row < g.y;
          if (!__any_sync(0xffffffffu, mine)) continue;
          const float sc = args.scales ? __ldg(args.scales + g.z) : 1.f;
          const uint32_t tb = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((acc * args.nb + i) * args.R);
          for (int c = 0; c < args.R; c += 16) {
            uint32_t v[16];
            tmem_ld16(tb + c, v);
            tmem_wait_ld();
            if (mine && S > 1) {  // this CTA's share of the columns, added below
              float4* p = (float4*)(sD + (quarter * 32 + lane) * args.R + c);
#pragma unroll
              for (int j = 0; j < 4; j++)
                p[j] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
            } else if (mine) {
              float q[16];
#pragma unroll
              for (int j = 0; j < 16; j++) q[j] = c + j < args.rank ? sc * __uint_as_float(v[j]) : 0.f;
              store_q(args.job[it.job], row, args.R, c, q);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
  }
  if (threadIdx.x == 0 && *abort) {  // after a timeout, let copies still in flight land before the CTA exits
    const uint64_t t0 = gtimer();
    while (gtimer() - t0 < 1000000ull) {}
  }
  tc_fence_before();
  if (S > 1) {
    cluster_sync();
    // one item per cluster: rank r adds rows [r·128/S, (r+1)·128/S) of all the CTAs' shares
    const int t = first >= args.ntiles ? first - args.ntiles : first, m0 = t * BM, rows = BM / S;
    const int2 segs = __ldg(args.tiles + t);
    const ShrinkJob& job = args.job[first >= args.ntiles];
    for (int lr = rank * rows + (int)threadIdx.x / 16; lr < (rank + 1) * rows; lr += TC_THREADS / 16) {
      const int row = m0 + lr;
      int a = -1;
      for (int s = 0; s < segs.y; s++) {
        const int4 g = __ldg(&args.segs[segs.x + s]);
        if (row >= g.x && row < g.y) a = g.z;
      }
      if (a < 0) continue;
      const float sc = args.scales ? __ldg(args.scales + a) : 1.f;
      for (int c = threadIdx.x & 15; c < args.R; c += 16) {
        const uint32_t at = smem_u32(sD + lr * args.R + c);
        float v = 0.f;
        for (int q = 0; q < S; q++) v += ld_cluster_f32(mapa_rank(at, (uint32_t)q));
        const float q[1] = {c < args.rank ? sc * v : 0.f};
        store_q(job, row, args.R, c, q);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its shared memory
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, args.tmem_cols);
  }
}

// ------------------------------------------------------------- outer
//
// D [columns of X, N] += X-blockᵀ · Q-block over blocks of up to 64 rows of one
// adapter and 256 columns (two M = 128 accumulators, so that Q and the steps of
// a block are shared by twice the columns): both operands are read MN-major from the row-major blocks that
// TMA brings (their rows are the contraction). N covers the three parts of Q
// (bf16) or the four of H (f16) of up to 64 rank rows, side by side; the
// epilogue adds them, each times its unit, smallest first. A block
// that ends inside its adapter's rows is loaded up to the next multiple of 16
// rows, which may be another request's: a warp of its own writes zeros over
// those before the MMA reads them (a product with zero would let an inf or NaN
// of that request through).
//
// The work is the blocks of all adapters, in adapter order, once for every tile
// (256 columns of one of the products and one group of 64 rank rows), tile
// after tile; every CTA takes an equal run of it. The blocks of an adapter
// that lie in one run are summed there and stored; of an adapter that several
// runs share, each run stores an f32 partial (at most two to a run, one where
// it begins and one where it ends), and k_outer_join adds them in the order of
// the runs: the same bits every time. (One CTA adding them, the last to
// arrive, took longer than the products: 150 us for one adapter of rank 64
// over 24 runs.)
//
// Bound by the read of X: 69,135 rows of 2304 and of 768 columns in f16 (424
// MB), rank 16, take 82 us with 256 requests (5.2 TB/s); 40,000 of 5248 and of
// 1024 in bf16, rank 32, 123 us. Equal runs: with a whole number of runs per
// tile (125 of 148 SMs) the latter took 8 us more.
constexpr int OUTER_THREADS = TC_THREADS + 32;  // and the warp that clears rows
constexpr int BC = 256;                         // columns of X per CTA
constexpr uint32_t XC_BYTES = 64 * BC * 2;
struct OuterJob {
  CUtensorMap tmX, tmQ, tmX16, tmQ16;  // boxes of 64 and of 16 rows
  int whole;                           // the maps of X bring this many 64-column blocks at once (3-D maps); 0: one at a time
  void* dP;
  int C, ctiles;
};
struct OuterArgs {
  OuterJob job[2];
  int rank, nchunks, ntiles, qstep, rgroups, nmma, stages, naccs;  // qstep: columns from one box of Q to the next
  uint32_t q_bytes, tmem_cols;
  const int4* chunks;  // row0, rows, adapter
  const int32_t* chunk_ptr;
  float* part;         // [runs, 2, rank rows of a tile, 256]
};

struct OuterTile {
  int job, c0, j0;       // product, first column, first rank row
  int xblocks, halves;   // 64-column blocks of X, accumulators of 128 columns
  __device__ OuterTile(const OuterArgs& args, int t) {
    const int ct = t / args.rgroups;
    job = ct >= args.job[0].ctiles;
    c0 = (job ? ct - args.job[0].ctiles : ct) * BC;
    j0 = (t % args.rgroups) * 64;
    xblocks = min(BC / 64, (args.job[job].C - c0 + 63) / 64);
    halves = xblocks > 2 ? 2 : 1;
  }
};

template <typename T> struct OuterParts;  // how Q is held beside an X of type T
template <> struct OuterParts<__nv_bfloat16> {
  static constexpr int n = kQParts;
  __device__ static float unit(int) { return 1.f; }
};
template <> struct OuterParts<__half> {
  static constexpr int n = kHParts;
  __device__ static float unit(int k) { return k == 0 ? 0x1p19f : k == 1 ? 0x1p8f : k == 2 ? 0x1p-3f : 0x1p-14f; }
};

template <typename T>
__global__ void __launch_bounds__(OUTER_THREADS, 1) k_outer_tc(const __grid_constant__ OuterArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t stage_bytes = XC_BYTES + args.q_bytes;
  uint64_t* full = (uint64_t*)(smem + args.stages * stage_bytes);
  uint64_t* empty = full + args.stages;
  uint64_t* cleared = empty + args.stages;
  uint64_t* tfull = cleared + args.stages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = (uint32_t*)(tempty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t total = (int64_t)args.ntiles * args.nchunks, lo = blockIdx.x * total / gridDim.x, hi = (blockIdx.x + 1) * total / gridDim.x;
  const int qblocks = (int)(args.q_bytes >> 13);  // 64-column blocks of Q
  if (threadIdx.x == 0) {
    for (int s = 0; s < args.stages; s++) mbar_init(&full[s], 1), mbar_init(&empty[s], 1), mbar_init(&cleared[s], 1);
    for (int a = 0; a < 2; a++) mbar_init(&tfull[a], 1), mbar_init(&tempty[a], 4);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(tmem_slot, args.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, used = 0, last_phase = 0;
      OuterTile t(args, (int)(lo / args.nchunks));
      int c = (int)(lo % args.nchunks);
      int4 ahead = __ldg(&args.chunks[c]);
      for (int64_t f = lo; f < hi; f++) {
        const int4 ch = ahead;
        if (++c == args.nchunks) c = 0;
        if (f + 1 < hi) ahead = __ldg(&args.chunks[c]);
        const OuterJob& job = args.job[t.job];
        const int c0 = t.c0, j0 = t.j0, xblocks = t.xblocks;
        if (!mbar_wait(&empty[stage], phase ^ 1, abort, &g_adapter_err)) break;
        uint8_t* st = smem + stage * stage_bytes;
        const int n16 = (ch.y + 15) >> 4;
        mbar_arrive_expect_tx(&full[stage], (uint32_t)(((job.whole ? job.whole : xblocks) + qblocks) * n16) * 2048);
        // X: whole blocks of 64 x 64 one after the other; where the rows end
        // earlier, 16 rows of all columns after 16 rows
        const int groups = n16 == 4 ? 1 : n16, high = n16 == 4 ? 8192 : 2048;
        const CUtensorMap *mx = n16 == 4 ? &job.tmX : &job.tmX16, *mq = n16 == 4 ? &job.tmQ : &job.tmQ16;
#pragma unroll 1
        for (int i = 0; i < groups; i++) {
          if (job.whole) {
            tma_load_3d(st + i * 8192, mx, &full[stage], 0, ch.x + 16 * i, c0 / 64);
          } else {
#pragma unroll 1
            for (int b = 0; b < xblocks; b++) tma_load_2d(st + i * 8192 + b * high, mx, &full[stage], c0 + 64 * b, ch.x + 16 * i);
          }
#pragma unroll 1
          for (int b = 0; b < qblocks; b++)
            tma_load_2d(st + XC_BYTES + b * 8192 + i * 2048, mq, &full[stage], b * args.qstep + j0, ch.x + 16 * i);
        }
        used |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == args.stages) { stage = 0; phase ^= 1; }
        if (c == 0 && f + 1 < hi) t = OuterTile(args, (int)((f + 1) / args.nchunks));
      }
      for (int s = 0; s < args.stages; s++)
        if (used >> s & 1) {
          const uint64_t t0 = gtimer();
          while (!mbar_try_wait(&full[s], (last_phase >> s) & 1) && gtimer() - t0 < kWaitNs) {}
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_rt<T>(args.nmma, true, true);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      uint64_t* last = nullptr;
      uint32_t last_phase = 0;
      for (int64_t f = lo; f < hi && ok;) {  // the pieces of the run: blocks of one adapter for one tile
        const int halves = OuterTile(args, (int)(f / args.nchunks)).halves;
        int c = (int)(f % args.nchunks);
        const int a = __ldg(&args.chunks[c].z), begin = c, end = (int)min(c + hi - f, (int64_t)__ldg(args.chunk_ptr + a + 1));
        f += end - begin;
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort, &g_adapter_err)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * 2 * args.nmma);
        for (; c < end; c++) {
          const int rows = __ldg(&args.chunks[c].y), steps = (rows + 15) >> 4;
          if (!mbar_wait(&full[stage], phase, abort, &g_adapter_err)) { ok = false; break; }
          if (!mbar_wait(&cleared[stage], phase, abort, &g_adapter_err)) { ok = false; break; }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + stage * stage_bytes), b0 = a0 + XC_BYTES;
          // (a last block of 64 columns or less: the other half of the accumulator's rows reads a stale block and is not stored)
          const uint32_t high = steps == 4 ? 8192 : 2048, step = steps == 4 ? 2048 : 8192;
          for (int k = 0; k < steps; k++) {
            const uint64_t q = sdesc_sw128_mn(b0 + k * 2048, 8192);
            tc_mma(d, sdesc_sw128_mn(a0 + k * step, high), q, idesc, (c > begin || k > 0) ? 1u : 0u);
            if (halves == 2) tc_mma(d + args.nmma, sdesc_sw128_mn(a0 + 2 * high + k * step, high), q, idesc, (c > begin || k > 0) ? 1u : 0u);
          }
          tc_commit(&empty[stage]);
          last = &empty[stage];
          last_phase = phase;
          if (++stage == args.stages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull[acc]);
        last = &tfull[acc];
        last_phase = acc_phase;
        if (++acc == args.naccs) { acc = 0; acc_phase ^= 1; }
      }
      if (last) {
        const uint64_t t0 = gtimer();
        while (!mbar_try_wait(last, last_phase) && gtimer() - t0 < kWaitNs) {}
      }
    }
  } else if (warp == 6) {
    // clears the rows of a block that are not its adapter's; passes on every
    // block, so that it is never a whole turn of the ring ahead or behind
    int stage = 0;
    uint32_t phase = 0;
    OuterTile t(args, (int)(lo / args.nchunks));
    int c = (int)(lo % args.nchunks);
    for (int64_t f = lo; f < hi; f++) {
      const int rows = __ldg(&args.chunks[c].y), xblocks = t.xblocks;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort, &g_adapter_err))) break;
      if (rows & 15) {
        uint8_t* st = smem + stage * stage_bytes;
        const int zn = (16 - (rows & 15)) * 8;  // 16-byte pieces per 64-column block
        const int first = rows > 48 ? rows * 128 : (rows >> 4) * 8192 + (rows & 15) * 128, high = rows > 48 ? 8192 : 2048;
        for (int k = 0; k < xblocks + qblocks; k++) {
          uint8_t* z = k < xblocks ? st + first + k * high : st + XC_BYTES + (k - xblocks) * 8192 + rows * 128;
          for (int i = lane; i < zn; i += 32) *(uint4*)(z + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&cleared[stage]);
      if (++stage == args.stages) { stage = 0; phase ^= 1; }
      if (++c == args.nchunks) {
        c = 0;
        if (f + 1 < hi) t = OuterTile(args, (int)((f + 1) / args.nchunks));
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    constexpr int NP = OuterParts<T>::n;
    const int nh = args.nmma / NP;  // rank rows of a tile, rounded up
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int64_t f = lo; f < hi;) {
      const int tt = (int)(f / args.nchunks), c = (int)(f % args.nchunks);
      const OuterTile t(args, tt);
      const OuterJob& job = args.job[t.job];
      const int64_t tile0 = (int64_t)tt * args.nchunks, size = (int64_t)args.rank * job.C;
      const int a = __ldg(&args.chunks[c].z), p0 = __ldg(args.chunk_ptr + a), p1 = __ldg(args.chunk_ptr + a + 1);
      const bool whole = tile0 + p0 >= lo && tile0 + p1 <= hi;
      float* part = args.part + (int64_t)(2 * blockIdx.x + (f == lo ? 0 : 1)) * nh * BC + quarter * 32 + lane;
      const int col0 = t.c0 + quarter * 32 + lane, j0 = t.j0, halves = t.halves;
      T* dP = (T*)job.dP;
      f = min(hi, tile0 + p1);
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, abort, &g_adapter_err))) break;
      tc_fence_after();
      for (int h = 0; h < halves; h++) {
        const int col = col0 + 128 * h;
        const uint32_t tb = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((acc * 2 + h) * args.nmma);
        for (int j = 0; j < nh; j += 16) {
          uint32_t v[NP][16];
#pragma unroll
          for (int k = 0; k < NP; k++) tmem_ld16(tb + k * nh + j, v[k]);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int row = j0 + j + i;
            if (row < args.rank && col < job.C) {
              float sum = OuterParts<T>::unit(NP - 1) * __uint_as_float(v[NP - 1][i]);
#pragma unroll
              for (int k = NP - 2; k >= 0; k--) sum = fmaf(OuterParts<T>::unit(k), __uint_as_float(v[k][i]), sum);
              if (whole) dP[a * size + (int64_t)row * job.C + col] = TcFmt<T>::cvt(sum);
              else part[(j + i) * BC + 128 * h] = sum;
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      if (++acc == args.naccs) { acc = 0; acc_phase ^= 1; }
    }
  }
  if (threadIdx.x == 0 && *abort) {
    const uint64_t t0 = gtimer();
    while (gtimer() - t0 < 1000000ull) {}
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, args.tmem_cols);
  }
}

// dP of the adapters that several runs share (the sum of their partials) and of
// those without rows (zeros). A thread per value, so the partials of one (148
// at most) are read in a row by neighbours; bound by latency, ~3 us.
constexpr int kMaxRuns = 256;
struct JoinArgs {
  const float* part;
  void* dP[2];
  int C[2], ctiles0, njobs;
  int rank, rgroups, nh, nshared, nempty;
  const int32_t* empty;
  int4 shared[kMaxRuns - 1];  // tile, adapter, slot of the first partial, number of partials: at most one per boundary
};
// grid: (rank rows of a group, shared adapters and then empty ones)
template <typename T>
__global__ void __launch_bounds__(BC) k_outer_join(const __grid_constant__ JoinArgs args) {
  pdl_wait();
  pdl_trigger();
  for (int e = blockIdx.y; e < args.nshared + args.nempty; e += gridDim.y) {
    if (e >= args.nshared) {
      const int64_t a = __ldg(args.empty + e - args.nshared);
      for (int j = 0; j < args.njobs; j++)
        for (int row = blockIdx.x; row < args.rank; row += gridDim.x)
          for (int col = threadIdx.x; col < args.C[j]; col += BC) ((T*)args.dP[j])[(a * args.rank + row) * args.C[j] + col] = from_f<T>(0.f);
      continue;
    }
    const int4 s = args.shared[e];
    const int ct = s.x / args.rgroups, j = ct >= args.ctiles0;
    const int col = (j ? ct - args.ctiles0 : ct) * BC + threadIdx.x, row = (s.x % args.rgroups) * 64 + blockIdx.x;
    const int64_t size = (int64_t)args.rank * args.C[j], at = (int64_t)row * args.C[j] + col;
    if (row >= args.rank || col >= args.C[j]) continue;
    // the first partial, and the one each of the next runs begins with
    const int64_t slot = (int64_t)args.nh * BC;
    float v = args.part[s.z * slot + blockIdx.x * BC + threadIdx.x];
    const float* p = args.part + (s.z / 2 + 1) * 2 * slot + blockIdx.x * BC + threadIdx.x;
#pragma unroll 8
    for (int i = 1; i < s.w; i++, p += 2 * slot) v += *p;
    ((T*)args.dP[j])[s.y * size + at] = from_f<T>(v);
  }
}

uint32_t tmem_columns(int want) {
  uint32_t c = 32;
  while ((int)c < want) c *= 2;
  return c;
}

template <typename T>
void shrink_t(const AdapterShrink* c, int njobs, const AdapterPlan& p, cudaStream_t st) {
  const int dtype = std::is_same<T, __half>::value ? LC_F16 : LC_BF16;
  ShrinkArgs a{};
  a.njobs = njobs;
  a.T = p.rows;
  a.ntiles = (p.rows + BM - 1) / BM;
  a.rank = c[0].rank;
  a.R = adapter_rank_rows(a.rank);
  // adapters side by side: four of 16 rank rows, two of 32 or 64 (a ragged tile
  // of 128 rows meets two or three requests), one above. The ring then has four
  // stages up to 32 rank rows, three up to 128 and two above (40,000 rows of
  // 1024 columns, both directions, bf16 / f16: rank 16 42 / 44 us, 64 54 / 64,
  // 128 81 / 96, 256 141 / 172)
  a.nb = a.R <= 32 ? 64 / a.R : a.R == 64 ? 2 : 1;
  a.bank_bytes = (uint32_t)(a.nb * a.R * 256);
  a.tmem_cols = tmem_columns(2 * a.nb * a.R);
  a.segs = p.segs;
  a.tiles = p.tiles;
  a.scales = c[0].scales;
  int KB = INT32_MAX;
  for (int j = 0; j < njobs; j++) {
    const AdapterShrink& q = c[njobs == 2 && c[1].C > c[0].C ? 1 - j : j];
    a.job[j].blocks = q.C % 64 == 0;
    a.job[j].tmX = a.job[j].blocks ? tensor_map_blocks(q.X, p.rows, q.C, q.ld, 2, BM, dtype) : tensor_map_2d(q.X, p.rows, q.C, q.ld, BK, BM, dtype);
    a.job[j].tmP = tensor_map_3d(q.P, q.n, q.rank, q.C, q.ldp, a.R, dtype);
    a.job[j].Q = q.Q;
    a.job[j].H = q.H;
    a.job[j].C = (int)q.C;
    KB = std::min(KB, (a.job[j].C + SK - 1) / SK);
  }
  const int64_t items = (int64_t)njobs * a.ntiles;
  a.S = 1;
  // a cluster's exchange costs ~2 us: split where it saves five stages at least
  // (0.4 us each; f16, rank 16: 8192 rows of 768, 6 stages, whole 9.7, in two
  // 11.4 us; 4096 rows of 1024, 8 stages, whole 10.6, in four 9.5 us)
  for (int f : {8, 4, 2})
    if (a.R <= 64 && items * f <= num_sms() && KB >= f && KB - KB / f >= 5) {
      a.S = f;
      break;
    }
  const int ctas = (int)std::min<int64_t>(items, num_sms());
  if (njobs == 2 && a.S == 1 && a.ntiles % ctas) {
    a.extra = ((a.job[0].C + SK - 1) / SK) / ((a.job[1].C + SK - 1) / SK);
    a.filled = (int)std::min<int64_t>(a.ntiles, (int64_t)a.extra * (ctas - a.ntiles % ctas));
  }
  const size_t d_bytes = a.S > 1 ? (size_t)BM * a.R * 4 : 0;
  a.stages = std::min(8, (int)(((224u << 10) - d_bytes) / (X_BYTES + a.bank_bytes)));
  const size_t smem = (size_t)a.stages * (X_BYTES + a.bank_bytes) + d_bytes + 1024 + 512;
  static bool attr = false;
  if (!attr) {
    CUDA_OK(cudaFuncSetAttribute(k_shrink_tc<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 << 10));
    attr = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  int n = 0;
  if (a.S > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = a.S;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    n = 1;
  }
  cfg.gridDim = dim3((unsigned)(a.S > 1 ? a.S * items : ctas));
  cfg.blockDim = dim3(TC_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  chain_attrs(cfg, at, n);
  CUDA_OK(cudaLaunchKernelEx(&cfg, k_shrink_tc<T>, a));
  LC_LAUNCHED(1);
}

// The runs of an outer product's work: one per SM.
struct OuterRuns {
  int ntiles = 0, runs = 0;
  int64_t total = 0;
  OuterRuns(const AdapterOuter* c, int njobs, const AdapterPlan& p) {
    for (int j = 0; j < njobs; j++) ntiles += (int)((c[j].C + BC - 1) / BC) * std::max(1, adapter_rank_rows(c[j].rank) / 64);
    total = (int64_t)ntiles * p.nchunks;
    runs = (int)std::min<int64_t>(std::min(num_sms(), kMaxRuns), total);
  }
};

template <typename T>
void outer_t(const AdapterOuter* c, int njobs, float* part, const AdapterPlan& p, cudaStream_t st) {
  const int dtype = std::is_same<T, __half>::value ? LC_F16 : LC_BF16;
  OuterArgs a{};
  a.rank = c[0].rank;
  a.nchunks = p.nchunks;
  constexpr int NP = OuterParts<T>::n;
  const int R = adapter_rank_rows(a.rank), nh = std::min(R, 64), qcols = NP * R;
  a.rgroups = std::max(1, R / 64);
  a.nmma = NP * nh;
  a.qstep = std::max(R, 64);
  a.q_bytes = (uint32_t)((a.nmma + 63) / 64 * 8192);
  a.stages = std::min(5, (int)((224u << 10) / (XC_BYTES + a.q_bytes)));
  // two accumulators, each of two halves of the columns, where TMEM's 512 columns hold them (up to 32 rank rows)
  a.naccs = 4 * a.nmma <= 512 ? 2 : 1;
  a.tmem_cols = tmem_columns(2 * a.naccs * a.nmma);
  a.chunks = p.chunks;
  a.chunk_ptr = p.chunk_ptr;
  const OuterRuns runs(c, njobs, p);
  a.ntiles = runs.ntiles;
  a.part = part;
  for (int j = 0; j < njobs; j++) {
    OuterJob& o = a.job[j];
    o.C = (int)c[j].C;
    o.ctiles = (o.C + BC - 1) / BC;
    // columns as blocks of 64, when they are: one load brings the blocks of a CTA, each 64 rows of 128 bytes
    o.whole = c[j].C % 64 == 0 ? (int)std::min<int64_t>(BC, c[j].C) / 64 : 0;
    o.tmX = o.whole ? tensor_map_blocks(c[j].X, p.rows, c[j].C, c[j].ld, o.whole, 64, dtype)
                    : tensor_map_2d(c[j].X, p.rows, c[j].C, c[j].ld, 64, 64, dtype);
    o.tmQ = tensor_map_2d(c[j].parts, p.rows, qcols, qcols, 64, 64, dtype);
    o.tmX16 = o.whole ? tensor_map_blocks(c[j].X, p.rows, c[j].C, c[j].ld, o.whole, 16, dtype)
                      : tensor_map_2d(c[j].X, p.rows, c[j].C, c[j].ld, 64, 16, dtype);
    o.tmQ16 = tensor_map_2d(c[j].parts, p.rows, qcols, qcols, 64, 16, dtype);
    o.dP = c[j].dP;
  }
  const size_t smem = (size_t)a.stages * (XC_BYTES + a.q_bytes) + 1024 + 512;
  static bool attr = false;
  if (!attr) {
    CUDA_OK(cudaFuncSetAttribute(k_outer_tc<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 << 10));
    attr = true;
  }
  launch_chain(k_outer_tc<T>, dim3((unsigned)runs.runs), dim3(OUTER_THREADS), smem, st, a);
  LC_LAUNCHED(1);
  JoinArgs join{};
  for (int i = 1; i < runs.runs; i++) {
    const int64_t f = i * runs.total / runs.runs;  // where run i begins
    const int tile = (int)(f / p.nchunks), at = (int)(f % p.nchunks);
    const int ad = (int)(std::upper_bound(p.host_chunk_ptr.begin(), p.host_chunk_ptr.end(), at) - p.host_chunk_ptr.begin()) - 1;
    if (p.host_chunk_ptr[ad] == at) continue;  // with an adapter
    int4* last = join.nshared ? &join.shared[join.nshared - 1] : nullptr;
    if (last && last->x == tile && last->y == ad) {
      last->w++;
    } else {  // run i - 1 ends with it, unless it is all of that run
      const bool begins = (int64_t)tile * p.nchunks + p.host_chunk_ptr[ad] == (i - 1) * runs.total / runs.runs;
      join.shared[join.nshared++] = make_int4(tile, ad, 2 * (i - 1) + (begins ? 0 : 1), 2);
    }
  }
  if (!join.nshared && !p.nempty) return;
  join.nempty = p.nempty;
  join.empty = p.empty;
  join.rank = a.rank;
  join.rgroups = a.rgroups;
  join.njobs = njobs;
  join.ctiles0 = a.job[0].ctiles;
  join.nh = nh;
  join.part = part;
  for (int j = 0; j < njobs; j++) {
    join.dP[j] = a.job[j].dP;
    join.C[j] = a.job[j].C;
  }
  launch_chain(k_outer_join<T>, dim3((unsigned)std::min(a.rank, 64), (unsigned)std::min(join.nshared + p.nempty, 65535)), dim3(BC), 0, st, join);
  LC_LAUNCHED(1);
}

}  // namespace

namespace lc {

// Reading the error word costs every flush a blocking copy (~15 us): it is
// read once a kernel of this file has been launched or recorded.
static bool launched = false;

void adapter_shrink_tc(const AdapterShrink* c, int njobs, const AdapterPlan& p, int dtype, cudaStream_t st) {
  if (!p.nsegs) return;
  launched = true;
  dtype == LC_F16 ? shrink_t<__half>(c, njobs, p, st) : shrink_t<__nv_bfloat16>(c, njobs, p, st);
}

size_t adapter_part_bytes(const AdapterOuter* c, int njobs, const AdapterPlan& p) {
  const OuterRuns runs(c, njobs, p);
  return (size_t)runs.runs * 2 * std::min(adapter_rank_rows(c[0].rank), 64) * BC * 4;
}

void adapter_outer_tc(const AdapterOuter* c, int njobs, void* part, const AdapterPlan& p, int dtype, cudaStream_t st) {
  launched = true;
  dtype == LC_F16 ? outer_t<__half>(c, njobs, (float*)part, p, st) : outer_t<__nv_bfloat16>(c, njobs, (float*)part, p, st);
}

std::string take_adapter_errors() {
  if (!launched) return "";
  unsigned int e = 0, z = 0;
  CUDA_OK(cudaMemcpyFromSymbol(&e, g_adapter_err, sizeof(e)));
  if (!e) return "";
  CUDA_OK(cudaMemcpyToSymbol(g_adapter_err, &z, sizeof(z)));
  return "adapters: a pipeline wait timed out (kernel aborted its tile loop)";
}

}  // namespace lc

// Sets this unit's bounded-wait limit (lc_debug_set_wait_limit).
void lc_internal_wait_limit_adapters(unsigned long long ns) { CUDA_OK(cudaMemcpyToSymbol(sm100::g_wait_limit_ns, &ns, sizeof(ns))); }
