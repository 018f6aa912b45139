// The adapter operators on few rows (f16 and bf16): dot products on the CUDA
// cores, where a tensor-core kernel would spend longer setting up its pipeline
// than computing.
//
// Both products are one: 8 rows of X against 16 rows of a matrix P whose long
// axis is contiguous. A block of 8 warps takes such a piece: warp w the four P
// rows of group w % 4 over one half of the columns (w / 4), 16-byte loads, 32
// f32 pair sums per lane, which a halving exchange reduces over the warp (31
// shuffles leave result l in lane l) and shared memory over the two halves.
//   shrink  8 rows of one request against its adapter's rank rows -> Q
//   linear  8 rows of the batch against 16 rows of W, plus bias and each row's
//           own Q · P_a
// Bound by latency and, with few rows, the read of W (or the bank) from L2: 8
// rows of 8 tenants, 768 -> 2304 in bf16, rank 16, take 3.2 + 5.1 us (3.5 MB
// of W); one launch instead of two, with u shared over a cluster, took 12.8.
// 234 and 252 registers keep one block on an SM: held to 128 they spill, and
// the pair took 3 us more.
#include "lc_adapters.h"
#include "lc_api.h"
#include "lc_gemm.h"
#include "lc_sm100.cuh"

#include <algorithm>

namespace {
using namespace lc;
using sm100::fma2;

constexpr int ROWS = 8, COLS = 16, THREADS = 256;

template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t u) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*(const __half2*)&u);
  else return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Lane l's result of the block's warps: row l % 8 of X against P row 4·(warp % 4) + l / 8. Rows from nx
// and from np on are not read (and give nothing that is used). `red` holds 128 floats.
template <typename T>
__device__ __forceinline__ float dot_piece(const T* X, int64_t ldx, int nx, const T* P, int64_t ldp, int np, int C, float* red) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j0 = (warp & 3) * 4, half = warp >> 2;
  float2 acc[4][ROWS];
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int i = 0; i < ROWS; i++) acc[j][i] = make_float2(0.f, 0.f);
  if (j0 < np) {
#pragma unroll 2
    for (int c = (half * 32 + lane) * 8; c < C; c += 512) {
      uint4 p[4], x[ROWS];
#pragma unroll
      for (int j = 0; j < 4; j++) p[j] = j0 + j < np ? __ldg((const uint4*)(P + (j0 + j) * ldp + c)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < ROWS; i++)
        if (i < nx) x[i] = __ldg((const uint4*)(X + i * ldx + c));
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float2 pf[4];
#pragma unroll
        for (int j = 0; j < 4; j++) pf[j] = pair_of<T>((&p[j].x)[e]);
#pragma unroll
        for (int i = 0; i < ROWS; i++)
          if (i < nx) {
            const float2 xf = pair_of<T>((&x[i].x)[e]);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j][i] = fma2(xf, pf[j], acc[j][i]);
          }
      }
    }
  }
  // value 8·j + i to lane 8·j + i: each exchange halves the values a lane holds
  float v[32];
#pragma unroll
  for (int j = 0; j < 4; j++)
#pragma unroll
    for (int i = 0; i < ROWS; i++) v[8 * j + i] = acc[j][i].x + acc[j][i].y;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; i++) {
      const float send = up ? v[i] : v[i + o], keep = up ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  if (half) red[(warp & 3) * 32 + lane] = v[0];
  __syncthreads();
  return half ? 0.f : v[0] + red[(warp & 3) * 32 + lane];
}

struct RowsShrinkJob {
  const void *X, *P;
  __nv_bfloat16* Q;
  __half* H;
  int64_t ldx, ldp;
  int C;
};
struct RowsShrinkArgs {
  RowsShrinkJob job[2];
  int rank, R, npieces;
  const int4* pieces;  // up to 8 rows of one adapter
  const float* scales;
  BankSplit split;
};

// grid: (pieces and then blocks for the split, groups of 16 rank rows, jobs)
template <typename T>
__global__ void __launch_bounds__(THREADS, 1) k_shrink_rows(const __grid_constant__ RowsShrinkArgs args) {
  __shared__ float red[128];
  pdl_wait();
  pdl_trigger();  // after the wait: what runs before this kernel is done when the next one starts
  if (blockIdx.x >= args.npieces) {  // the blocks beside the pieces, of every group and job, in one range
    const int64_t nb = gridDim.x - args.npieces, b = blockIdx.x - args.npieces + nb * (blockIdx.y + (int64_t)gridDim.y * blockIdx.z);
    for (int64_t i = b * THREADS + threadIdx.x; i < args.split.steps; i += nb * gridDim.y * gridDim.z * THREADS) split_bank_step(args.split, i);
    return;
  }
  const RowsShrinkJob& job = args.job[blockIdx.z];
  const int4 pc = __ldg(&args.pieces[blockIdx.x]);
  const int j0 = blockIdx.y * COLS;
  const float v = dot_piece<T>((const T*)job.X + pc.x * job.ldx, job.ldx, pc.y, (const T*)job.P + ((int64_t)pc.z * args.rank + j0) * job.ldp,
                               job.ldp, args.rank - j0, job.C, red);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp >= 4) return;
  const int i = lane & 7, j = j0 + warp * 4 + (lane >> 3);
  if (i >= pc.y || j >= args.R) return;
  const float s = args.scales ? __ldg(args.scales + pc.z) : 1.f;
  const float q = j < args.rank ? s * v : 0.f;
  const int64_t t = (int64_t)pc.x + i;
  if (job.Q) {
    __nv_bfloat16 part[kQParts];
    split_bf16(q, part);
#pragma unroll
    for (int k = 0; k < kQParts; k++) job.Q[(t * kQParts + k) * args.R + j] = part[k];
  }
  if (job.H) {
    __half part[kHParts];
    split_f16(q, part);
#pragma unroll
    for (int k = 0; k < kHParts; k++) job.H[(t * kHParts + k) * args.R + j] = part[k];
  }
}

struct RowsLinearArgs {
  const void *x, *w, *bank, *bias;
  const __nv_bfloat16* Q;
  void* y;
  int64_t M, ldx, ldw, ldb, ldy;
  int N, K, rank, R, bias_dtype, defer, ngroups;  // ngroups: groups of 16 columns
  const int2* tiles;
  const int4* segs;
};

// grid: groups of 16 columns, for each group of 8 rows
template <typename T>
__global__ void __launch_bounds__(THREADS, 1) k_linear_rows(const __grid_constant__ RowsLinearArgs args) {
  __shared__ float red[128];
  if (!args.defer) pdl_wait();
  pdl_trigger();
  const int n0 = (int)(blockIdx.x % args.ngroups) * COLS;
  const int64_t t0 = (int64_t)(blockIdx.x / args.ngroups) * ROWS;
  float v = 0.f;
  if (args.w)
    v = dot_piece<T>((const T*)args.x + t0 * args.ldx, args.ldx, (int)min((int64_t)ROWS, args.M - t0), (const T*)args.w + n0 * args.ldw,
                     args.ldw, args.N - n0, args.K, red);
  pdl_wait();  // Q is written; and this kernel is not done before the ones it follows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = n0 + (warp & 3) * 4 + (lane >> 3);
  const int64_t t = t0 + (lane & 7);
  if (warp >= 4 || t >= args.M || n >= args.N) return;
  if (args.bias) v += ld_as<float>((const char*)args.bias, args.bias_dtype, n);
  const int a = adapter_of_row(args.tiles, args.segs, t);
  if (a >= 0) {
    const __nv_bfloat16* q = args.Q + t * kQParts * args.R;
    const T* p = (const T*)args.bank + (int64_t)a * args.rank * args.ldb + n;
    float d = 0.f;
#pragma unroll 8
    for (int j = 0; j < args.rank; j++) {
      const float u = __bfloat162float(q[j]) + (__bfloat162float(q[args.R + j]) + __bfloat162float(q[2 * args.R + j]));
      d = fmaf(u, to_f<T>(p[j * args.ldb]), d);
    }
    v += d;
  }
  ((T*)args.y)[t * args.ldy + n] = from_f<T>(v);
}

template <typename T>
void shrink_rows_t(const AdapterShrink* c, int njobs, const BankSplit& split, const AdapterPlan& p, cudaStream_t st) {
  RowsShrinkArgs a{};
  a.rank = c[0].rank;
  a.R = adapter_rank_rows(a.rank);
  a.npieces = p.npieces;
  a.pieces = p.pieces;
  a.split = split;
  a.scales = c[0].scales;
  for (int j = 0; j < njobs; j++) a.job[j] = {c[j].X, c[j].P, c[j].Q, c[j].H, c[j].ld, c[j].ldp, (int)c[j].ld};
  const int groups = (a.R + COLS - 1) / COLS, per = THREADS * groups * njobs;
  const unsigned beside = (unsigned)std::min<int64_t>((split.steps + per - 1) / per, 2 * num_sms());
  launch_chain(k_shrink_rows<T>, dim3((unsigned)p.npieces + beside, (unsigned)groups, (unsigned)njobs), dim3(THREADS), 0, st, a);
  LC_LAUNCHED(1);
}

template <typename T>
void linear_rows_t(const GemmAdaptedCall& c, const AdapterPlan& p, int rank, cudaStream_t st) {
  RowsLinearArgs a{};
  a.x = c.x;
  a.w = c.w;
  a.bank = c.share.bank;
  a.Q = (const __nv_bfloat16*)c.share.u;
  a.bias = c.bias;
  a.bias_dtype = c.bias_dtype;
  a.y = c.y;
  a.M = c.M;
  a.ldx = c.ldx;
  a.ldw = c.ldw;
  a.ldb = c.share.ld;
  a.ldy = c.ldy;
  a.N = (int)c.N;
  a.K = (int)c.ldx;  // rows of padded operands end in zeros
  a.rank = rank;
  a.R = c.share.R;
  a.defer = c.after_share ? 1 : 0;
  a.tiles = p.tiles;
  a.segs = p.segs;
  a.ngroups = (int)((c.N + COLS - 1) / COLS);
  launch_chain(k_linear_rows<T>, dim3((unsigned)(a.ngroups * ((c.M + ROWS - 1) / ROWS))), dim3(THREADS), 0, st, a);
  LC_LAUNCHED(1);
}

}  // namespace

namespace lc {

// Requests of 16 rows or less on average cost the tensor-core forms a pass each.
static int short_requests(const AdapterPlan& p) { return (int64_t)p.nsegs * 16 >= p.rows ? 2 : 1; }

bool adapter_shrink_rows_fit(const AdapterShrink* c, int njobs, const AdapterPlan& p) {
  int64_t C = 0;
  for (int j = 0; j < njobs; j++) C += c[j].ld;
  return p.npieces && (int64_t)p.rows * adapter_rank_rows(c[0].rank) * C <= kRowsShrinkMost * short_requests(p);
}

void adapter_shrink_rows(const AdapterShrink* c, int njobs, const BankSplit& split, const AdapterPlan& p, int dtype, cudaStream_t st) {
  dtype == LC_F16 ? shrink_rows_t<__half>(c, njobs, split, p, st) : shrink_rows_t<__nv_bfloat16>(c, njobs, split, p, st);
}

bool adapter_linear_rows_fit(int64_t M, int64_t N, int64_t K, const AdapterPlan& p) { return M * N * K <= kRowsLinearMost * short_requests(p); }

void adapter_linear_rows(const GemmAdaptedCall& c, const AdapterPlan& p, int rank, int dtype, cudaStream_t st) {
  dtype == LC_F16 ? linear_rows_t<__half>(c, p, rank, st) : linear_rows_t<__nv_bfloat16>(c, p, rank, st);
}

}  // namespace lc
