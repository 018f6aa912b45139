// The narrow products of the adapter operators on the tensor cores (f16 and
// bf16): the shrink Q[t, :] = s_a·P_a·X[t] and the outer sums
// dP_a = Σ_{t in a} Q[t] ⊗ X[t]. The wide product is gemm_adapted (lc_gemm.cu).
//
// Q is held as two 16-bit parts per value, high part and remainder, so that
// the tensor cores read it back as exactly as an f32 would be at the scale of
// the result (2^-16 of each value in bf16, 2^-22 in f16, 2^-25 absolute):
// [T, 2·R] with the high parts in columns [0, R), R = rank rounded up to 16
// (to 64 above 32). An f16 value beyond 65504 keeps its excess in the
// remainder, up to 131008.
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
constexpr uint32_t X_BYTES = BM * BK * 2;

template <typename T>
__device__ __forceinline__ uint32_t idesc_rt(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (TcFmt<T>::ab << 7) | (TcFmt<T>::ab << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
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
// The two 16-bit parts of a value.
template <typename T> __device__ __forceinline__ T largest();
template <> __device__ __forceinline__ __half largest<__half>() { return __ushort_as_half(0x7bff); }
template <> __device__ __forceinline__ __nv_bfloat16 largest<__nv_bfloat16>() { return __ushort_as_bfloat16(0x7f7f); }
template <typename T>
__device__ __forceinline__ void split2(float v, T& hi, T& lo) {
  hi = TcFmt<T>::cvt(v);
  float h = TcFmt<T>::back(hi);
  if (!isfinite(h)) {
    if (!isfinite(v)) {  // the value itself: its remainder would be NaN
      lo = TcFmt<T>::cvt(0.f);
      return;
    }
    h = copysignf(TcFmt<T>::back(largest<T>()), v);
    hi = TcFmt<T>::cvt(h);
  }
  lo = TcFmt<T>::cvt(v - h);
}

// ------------------------------------------------------------- shrink
//
// One CTA takes tiles of 128 rows. Per 64-column block of X the ring holds the
// X block (TMA, 16 KB) and, for up to `nb` of the tile's segments, the block of
// P_a (R rows); one MMA per segment and 16 columns adds to D [128, R] with the
// lanes outside the segment switched off, so every row meets its own adapter
// alone. More segments than nb: the tile's columns are streamed again.
// D is double-buffered in TMEM; the epilogue scales, splits and stores rows.
//
// Bound by the read of X. With few tiles the columns are split over clusters
// of S CTAs, whose partial D meet in shared memory and are added in rank order.
struct ShrinkArgs {
  int T, C, ntiles, nsegs, R, rank, nb, stages, ucols;
  uint32_t bank_bytes, tmem_cols;
  const int4* segs;
  const int32_t* tile_first;
  const int32_t* row_adapter;
  const float* scales;
  void* Q;
};

template <typename T>
__global__ void __launch_bounds__(TC_THREADS, 1) k_shrink_tc(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmP,
                                                             const __grid_constant__ ShrinkArgs args, int S) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t stage_bytes = X_BYTES + args.bank_bytes;
  uint64_t* full = (uint64_t*)(smem + args.stages * stage_bytes);
  uint64_t* empty = full + args.stages;
  uint64_t* tfull = empty + args.stages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = (uint32_t*)(tempty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int KB = (args.C + BK - 1) / BK, kb0 = (int)((int64_t)rank * KB / S), kb1 = (int)((int64_t)(rank + 1) * KB / S);
  const int first = blockIdx.x / S, step = gridDim.x / S;
  pdl_trigger();
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

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t used = 0, last_phase = 0;  // stages filled, and the phase bit of each one's last fill
      for (int t = first; t < args.ntiles && ok; t += step) {
        const int m0 = t * BM;
        for (int s = __ldg(args.tile_first + t); s < args.nsegs && ok; s += args.nb) {
          if (__ldg(&args.segs[s]).x >= m0 + BM) break;
          int n = 1;  // segments of this pass
          int ad[4];
          ad[0] = __ldg(&args.segs[s]).z;
#pragma unroll
          for (int i = 1; i < 4; i++) {
            ad[i] = 0;
            if (i < args.nb && n == i && s + i < args.nsegs) {
              const int4 g = __ldg(&args.segs[s + i]);
              if (g.x < m0 + BM) ad[i] = g.z, n = i + 1;
            }
          }
          for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&empty[stage], phase ^ 1, abort, &g_adapter_err)) { ok = false; break; }
            uint8_t* st = smem + stage * stage_bytes;
            mbar_arrive_expect_tx(&full[stage], X_BYTES + (uint32_t)n * args.R * 128);
            tma_load_2d(st, &tmX, &full[stage], kb * BK, m0);
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (i < n) tma_load_3d(st + X_BYTES + i * args.R * 128, &tmP, &full[stage], kb * BK, 0, ad[i]);
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
      const uint32_t idesc = idesc_rt<T>(args.R, false, false);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      uint64_t* last = nullptr;
      uint32_t last_phase = 0;
      for (int t = first; t < args.ntiles && ok; t += step) {
        const int m0 = t * BM;
        int s = __ldg(args.tile_first + t);
        if (s >= args.nsegs || __ldg(&args.segs[s]).x >= m0 + BM) continue;
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort, &g_adapter_err)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * args.R);
        for (; s < args.nsegs && ok; s += args.nb) {
          if (__ldg(&args.segs[s]).x >= m0 + BM) break;
          uint32_t off[4][4];
          int n = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (i < args.nb && n == i && s + i < args.nsegs) {
              const int4 g = __ldg(&args.segs[s + i]);
              if (g.x < m0 + BM) {
                n = i + 1;
#pragma unroll
                for (int w = 0; w < 4; w++) off[i][w] = lanes_off(m0 + 32 * w, g.x, g.y);
              }
            }
          }
          for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&full[stage], phase, abort, &g_adapter_err)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a0 = smem_u32(smem + stage * stage_bytes), b0 = a0 + X_BYTES;
#pragma unroll
            for (int i = 0; i < 4; i++)
              if (i < n)
#pragma unroll
                for (int k = 0; k < BK / 16; k++)
                  tc_mma_lanes(d, sdesc_sw128(a0 + k * 32), sdesc_sw128(b0 + i * args.R * 128 + k * 32), idesc, (kb > kb0 || k > 0) ? 1u : 0u, off[i]);
            tc_commit(&empty[stage]);
            last = &empty[stage];
            last_phase = phase;
            if (++stage == args.stages) { stage = 0; phase ^= 1; }
          }
        }
        if (!ok) break;
        tc_commit(&tfull[acc]);
        last = &tfull[acc];
        last_phase = acc_phase;
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
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
    T* Q = (T*)args.Q;
    for (int t = first; t < args.ntiles; t += step) {
      const int m0 = t * BM, s0 = __ldg(args.tile_first + t);
      if (s0 >= args.nsegs || __ldg(&args.segs[s0]).x >= m0 + BM) continue;
      const int row = m0 + quarter * 32 + lane;
      const int a = row < args.T ? __ldg(args.row_adapter + row) : -1;
      const float sc = a >= 0 && args.scales ? __ldg(args.scales + a) : 1.f;
      if (!mbar_wait(&tfull[acc], acc_phase, abort, &g_adapter_err)) break;
      tc_fence_after();
      const uint32_t tb = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * args.R);
      const int half = args.ucols / 2;
      for (int c = 0; c < args.R; c += 16) {
        uint32_t v[16];
        tmem_ld16(tb + c, v);
        tmem_wait_ld();
        if (S > 1) {  // this CTA's share of the columns: to shared memory, added below
          float* p = (float*)smem + (quarter * 32 + lane) * args.R + c;
#pragma unroll
          for (int j = 0; j < 16; j++) p[j] = __uint_as_float(v[j]);
          continue;
        }
        T hi[16], lo[16];
#pragma unroll
        for (int j = 0; j < 16; j++) split2<T>(c + j < args.rank ? sc * __uint_as_float(v[j]) : 0.f, hi[j], lo[j]);
        if (a >= 0) {
          uint4* ph = (uint4*)(Q + (int64_t)row * args.ucols + c);
          uint4* pl = (uint4*)(Q + (int64_t)row * args.ucols + half + c);
          ph[0] = ((const uint4*)hi)[0];
          ph[1] = ((const uint4*)hi)[1];
          pl[0] = ((const uint4*)lo)[0];
          pl[1] = ((const uint4*)lo)[1];
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  }
  if (threadIdx.x == 0 && *abort) {  // after a timeout, let copies still in flight land before the CTA exits
    const uint64_t t0 = gtimer();
    while (gtimer() - t0 < 1000000ull) {}
  }
  tc_fence_before();
  if (S > 1) {
    cluster_sync();
    // rank r adds rows [r·128/S, (r+1)·128/S) of all the CTAs' shares
    const int m0 = first * BM, rows = BM / S;
    T* Q = (T*)args.Q;
    for (int e = threadIdx.x; e < rows * args.R; e += TC_THREADS) {
      const int lr = rank * rows + e / args.R, c = e % args.R, row = m0 + lr;
      const int a = row < args.T ? __ldg(args.row_adapter + row) : -1;
      if (a < 0) continue;
      const uint32_t at = smem_u32(smem) + (uint32_t)(lr * args.R + c) * 4;
      float v = 0.f;
      for (int q = 0; q < S; q++) v += ld_cluster_f32(mapa_rank(at, (uint32_t)q));
      T hi, lo;
      split2<T>(c < args.rank ? (args.scales ? __ldg(args.scales + a) : 1.f) * v : 0.f, hi, lo);
      Q[(int64_t)row * args.ucols + c] = hi;
      Q[(int64_t)row * args.ucols + args.ucols / 2 + c] = lo;
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
// D [128 columns of X, N] += X-blockᵀ · Q-block over blocks of up to 64 rows of
// one adapter: both operands are read MN-major from the row-major blocks that
// TMA brings (their rows are the contraction). N covers the high and the
// remainder parts of up to 64 rank rows; the epilogue adds the two. A block
// that ends inside its adapter's rows loads rows of other requests too: the
// MMA warp writes zeros over them, up to the next multiple of 16, before the
// MMA reads them, and issues no steps past that.
//
// The blocks of all adapters, in adapter order, are cut into G equal runs; a
// CTA takes one run for one 128-column tile (and one group of 64 rank rows).
// A run that holds all of an adapter's blocks stores dP; otherwise it stores
// an f32 partial, in slot run + adapter (distinct for every pair that
// occurs), and k_outer_join adds an adapter's partials in the order of the
// runs: the same bits every time, without atomics. Bound by the read of X.
struct OuterArgs {
  int C, rank, nchunks, n, G, ucols, rgroups, nmma, stages;
  uint32_t q_bytes, tmem_cols;
  const int4* chunks;     // row0, rows, adapter
  const int32_t* chunk_ptr;
  float* part;
  void* dP;
};

template <typename T>
__global__ void __launch_bounds__(TC_THREADS, 1) k_outer_tc(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmQ,
                                                            const __grid_constant__ OuterArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t stage_bytes = X_BYTES + args.q_bytes;
  uint64_t* full = (uint64_t*)(smem + args.stages * stage_bytes);
  uint64_t* empty = full + args.stages;
  uint64_t* tfull = empty + args.stages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = (uint32_t*)(tempty + 2);
  volatile int* abort = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = blockIdx.x * BM, g = blockIdx.y, j0 = blockIdx.z * 64;
  const int lo = (int)((int64_t)g * args.nchunks / args.G), hi = (int)((int64_t)(g + 1) * args.nchunks / args.G);
  pdl_trigger();
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

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, used = 0, last_phase = 0;
      for (int c = lo; c < hi; c++) {
        const int row0 = __ldg(&args.chunks[c]).x;
        if (!mbar_wait(&empty[stage], phase ^ 1, abort, &g_adapter_err)) break;
        uint8_t* st = smem + stage * stage_bytes;
        mbar_arrive_expect_tx(&full[stage], stage_bytes);
        tma_load_2d(st, &tmX, &full[stage], c0, row0);
        tma_load_2d(st + 8192, &tmX, &full[stage], c0 + 64, row0);
        tma_load_2d(st + X_BYTES, &tmQ, &full[stage], j0, row0);
        if (args.q_bytes > 8192) tma_load_2d(st + X_BYTES + 8192, &tmQ, &full[stage], args.ucols / 2 + j0, row0);
        used |= 1u << stage;
        last_phase = (last_phase & ~(1u << stage)) | (phase << stage);
        if (++stage == args.stages) { stage = 0; phase ^= 1; }
      }
      for (int s = 0; s < args.stages; s++)
        if (used >> s & 1) {
          const uint64_t t0 = gtimer();
          while (!mbar_try_wait(&full[s], (last_phase >> s) & 1) && gtimer() - t0 < kWaitNs) {}
        }
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_rt<T>(args.nmma, true, true);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    uint64_t* last = nullptr;
    uint32_t last_phase = 0;
    for (int c = lo; c < hi && ok;) {
      const int a = __ldg(&args.chunks[c]).z, end = min(hi, __ldg(args.chunk_ptr + a + 1)), begin = c;
      if (!__all_sync(0xffffffffu, mbar_wait(&tempty[acc], acc_phase ^ 1, abort, &g_adapter_err))) { ok = false; break; }
      tc_fence_after();
      const uint32_t d = tmem + (uint32_t)(acc * args.nmma);
      for (; c < end; c++) {
        const int rows = __ldg(&args.chunks[c]).y, steps = (rows + 15) >> 4;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, abort, &g_adapter_err))) { ok = false; break; }
        uint8_t* st = smem + stage * stage_bytes;
        if (rows & 15) {  // rows of other requests in the last step: zeros in both operands
          const int z0 = rows * 128, zn = (steps * 16 - rows) * 8;  // 16-byte pieces per 64-column block
          const int blocks = (int)(stage_bytes >> 13);
          for (int i = lane; i < zn * blocks; i += 32) *(uint4*)(st + (i / zn) * 8192 + z0 + (i % zn) * 16) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t a0 = smem_u32(st), b0 = a0 + X_BYTES;
          for (int k = 0; k < steps; k++)
            tc_mma(d, sdesc_sw128_mn(a0 + k * 2048, 8192), sdesc_sw128_mn(b0 + k * 2048, 8192), idesc, (c > begin || k > 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
        }
        __syncwarp();
        last = &empty[stage];
        last_phase = phase;
        if (++stage == args.stages) { stage = 0; phase ^= 1; }
      }
      if (!ok) break;
      if (lane == 0) tc_commit(&tfull[acc]);
      __syncwarp();
      last = &tfull[acc];
      last_phase = acc_phase;
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (last) {
      const uint64_t t0 = gtimer();
      while (!mbar_try_wait(last, last_phase) && gtimer() - t0 < kWaitNs) {}
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, col = c0 + quarter * 32 + lane;
    const int nh = args.nmma / 2;  // rank rows of this CTA, rounded up
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int c = lo; c < hi;) {
      const int a = __ldg(&args.chunks[c]).z, p0 = __ldg(args.chunk_ptr + a), p1 = __ldg(args.chunk_ptr + a + 1);
      const bool whole = p0 >= lo && p1 <= hi;
      if (!mbar_wait(&tfull[acc], acc_phase, abort, &g_adapter_err)) break;
      tc_fence_after();
      const uint32_t tb = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * args.nmma);
      for (int j = 0; j < nh; j += 16) {
        uint32_t vh[16], vl[16];
        tmem_ld16(tb + j, vh);
        tmem_ld16(tb + nh + j, vl);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const int row = j0 + j + i;
          if (row < args.rank && col < args.C) {
            const float v = __uint_as_float(vh[i]) + __uint_as_float(vl[i]);
            if (whole) ((T*)args.dP)[((int64_t)a * args.rank + row) * args.C + col] = TcFmt<T>::cvt(v);
            else args.part[((int64_t)(g + a) * args.rank + row) * args.C + col] = v;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      c = min(hi, p1);
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

// dP of the adapters whose blocks lie in several runs (the sum of their
// partials) or that have no blocks (zeros).
template <typename T>
__global__ void __launch_bounds__(256) k_outer_join(const float* __restrict__ part, const int32_t* __restrict__ chunk_ptr, T* __restrict__ dP,
                                                    int nchunks, int G, int64_t size) {
  pdl_trigger();
  pdl_wait();
  const int a = blockIdx.y, p0 = chunk_ptr[a], p1 = chunk_ptr[a + 1];
  int g0 = 0, g1 = -1;
  if (p1 > p0) {  // the runs of the first and the last block: run g begins at floor(g·nchunks / G)
    g0 = (int)((((int64_t)p0 + 1) * G - 1) / nchunks);
    g1 = (int)(((int64_t)p1 * G - 1) / nchunks);
    if (g0 == g1) return;
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
    float v = 0.f;
    for (int g = g0; g <= g1; g++) v += part[(int64_t)(g + a) * size + i];
    dP[(int64_t)a * size + i] = from_f<T>(v);
  }
}

uint32_t tmem_columns(int want) {
  uint32_t c = 32;
  while ((int)c < want) c *= 2;
  return c;
}

template <typename T>
void shrink_t(const AdapterShrink& c, const AdapterPlan& p, cudaStream_t st) {
  const int dtype = std::is_same<T, __half>::value ? LC_F16 : LC_BF16;
  ShrinkArgs a{};
  a.T = p.rows;
  a.C = (int)c.C;
  a.ntiles = (p.rows + BM - 1) / BM;
  a.nsegs = p.nsegs;
  a.rank = c.rank;
  a.R = adapter_u_cols(c.rank) / 2;
  a.nb = std::max(1, std::min(4, 64 / a.R));
  a.bank_bytes = (uint32_t)(a.nb * a.R * 128);
  a.stages = std::min(8, (int)((200u << 10) / (X_BYTES + a.bank_bytes)));
  a.ucols = adapter_u_cols(c.rank);
  a.tmem_cols = tmem_columns(2 * a.R);
  a.segs = p.segs;
  a.tile_first = p.tile_first;
  a.row_adapter = p.row_adapter;
  a.scales = c.scales;
  a.Q = c.Q;
  const CUtensorMap mx = tensor_map_2d(c.X, p.rows, c.C, c.ld, BK, BM, dtype);
  const CUtensorMap mp = tensor_map_3d(c.P, c.n, c.rank, c.C, c.ldp, a.R, dtype);
  const int KB = (a.C + BK - 1) / BK;
  int S = 1;
  for (int f : {8, 4, 2})
    if (a.ntiles * f <= num_sms() && KB >= 2 * f) {
      S = f;
      break;
    }
  const size_t smem = (size_t)a.stages * (X_BYTES + a.bank_bytes) + 1024 + 512;
  static bool attr = false;
  if (!attr) {
    CUDA_OK(cudaFuncSetAttribute(k_shrink_tc<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 << 10));
    attr = true;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  int n = 0;
  if (S > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = S;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    n = 1;
  }
  cfg.gridDim = dim3(S > 1 ? S * a.ntiles : std::min(a.ntiles, num_sms()));
  cfg.blockDim = dim3(TC_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  chain_attrs(cfg, at, n);
  CUDA_OK(cudaLaunchKernelEx(&cfg, k_shrink_tc<T>, mx, mp, a, S));
  LC_LAUNCHED(1);
}

template <typename T>
void outer_t(const AdapterOuter& c, const AdapterPlan& p, cudaStream_t st) {
  const int dtype = std::is_same<T, __half>::value ? LC_F16 : LC_BF16;
  const int64_t size = (int64_t)c.rank * c.C;
  OuterArgs a{};
  a.C = (int)c.C;
  a.rank = c.rank;
  a.nchunks = p.nchunks;
  a.n = p.n_adapters;
  a.ucols = adapter_u_cols(c.rank);
  a.rgroups = std::max(1, a.ucols / 128);
  a.nmma = std::min(a.ucols, 128);
  a.q_bytes = a.ucols > 64 ? 16384 : 8192;
  a.stages = a.q_bytes > 8192 ? 6 : 8;
  a.tmem_cols = tmem_columns(2 * a.nmma);
  a.chunks = p.chunks;
  a.chunk_ptr = p.chunk_ptr;
  a.dP = c.dP;
  const int ct = (int)((c.C + BM - 1) / BM) * a.rgroups, sms = num_sms();
  // runs: one wave of CTAs at least, and whole waves as far as 16 runs can make them
  int G = 1;
  double best = 0;
  for (int f = 1; f <= 64 && f <= p.nchunks; f++) {
    const int64_t ctas = (int64_t)ct * f, waves = (ctas + sms - 1) / sms;
    const double fill = (double)ctas / (double)(waves * sms);
    if (fill > best + 0.03) best = fill, G = f;
    if (waves > 2) break;
  }
  a.G = G;
  struct Partials {
    void* p = nullptr;
    ~Partials() { if (p) dfree(p); }
  } part;
  if (G > 1) part.p = dmalloc((size_t)(G + p.n_adapters) * size * 4);
  a.part = (float*)part.p;
  const CUtensorMap mx = tensor_map_2d(c.X, p.rows, c.C, c.ld, 64, 64, dtype);
  const CUtensorMap mq = tensor_map_2d(c.Q, p.rows, a.ucols, a.ucols, 64, 64, dtype);
  const size_t smem = (size_t)a.stages * (X_BYTES + a.q_bytes) + 1024 + 512;
  static bool attr = false;
  if (!attr) {
    CUDA_OK(cudaFuncSetAttribute(k_outer_tc<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 << 10));
    attr = true;
  }
  LC_CHECK(p.n_adapters <= 65535, "adapters: more than 65535 adapters");
  if (p.nchunks) {
    launch_chain(k_outer_tc<T>, dim3((unsigned)((c.C + BM - 1) / BM), (unsigned)G, (unsigned)a.rgroups), dim3(TC_THREADS), smem, st, mx, mq, a);
    LC_LAUNCHED(1);
  }
  launch_chain(k_outer_join<T>, dim3((unsigned)std::min<int64_t>((size + 1023) / 1024, 256), (unsigned)p.n_adapters), dim3(256), 0, st,
               (const float*)part.p, (const int32_t*)p.chunk_ptr, (T*)c.dP, p.nchunks, G, size);
  LC_LAUNCHED(1);
}

}  // namespace

namespace lc {

void adapter_shrink_tc(const AdapterShrink& c, const AdapterPlan& p, int dtype, cudaStream_t st) {
  if (!p.nsegs) return;
  dtype == LC_F16 ? shrink_t<__half>(c, p, st) : shrink_t<__nv_bfloat16>(c, p, st);
}

void adapter_outer_tc(const AdapterOuter& c, const AdapterPlan& p, int dtype, cudaStream_t st) {
  if (!p.n_adapters) return;
  dtype == LC_F16 ? outer_t<__half>(c, p, st) : outer_t<__nv_bfloat16>(c, p, st);
}

std::string take_adapter_errors() {
  unsigned int e = 0, z = 0;
  CUDA_OK(cudaMemcpyFromSymbol(&e, g_adapter_err, sizeof(e)));
  if (!e) return "";
  CUDA_OK(cudaMemcpyToSymbol(g_adapter_err, &z, sizeof(z)));
  return "adapters: a pipeline wait timed out (kernel aborted its tile loop)";
}

}  // namespace lc

// Sets this unit's bounded-wait limit (lc_debug_set_wait_limit).
void lc_internal_wait_limit_adapters(unsigned long long ns) { CUDA_OK(cudaMemcpyToSymbol(sm100::g_wait_limit_ns, &ns, sizeof(ns))); }
