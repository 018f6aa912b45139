// Internal definitions of the adapter operators (include/laya_cuda_adapters.h).
#pragma once
#include "lc_common.cuh"
#include "lc_gemm.h"

constexpr int kAdapterMaxRank = 256;

// Rows and adapters of one batch on the device (lc_adapter_plan_create).
struct AdapterPlan {
  int rows = 0, n_adapters = 0, nsegs = 0, nchunks = 0, nempty = 0, nused = 0, npieces = 0;
  int32_t* dev = nullptr;          // one allocation behind the arrays below
  int4* segs = nullptr;            // [nsegs]: row ranges with an adapter, ascending: lo, hi, adapter, its place in `used`
  int2* tiles = nullptr;           // per 128 rows: the first segment that meets them, and how many do
  int2* spans = nullptr;           // [nsegs]: the row ranges adapter by adapter, ascending within one
  int32_t* span_ptr = nullptr;     // [n_adapters + 1]: where each adapter's spans start
  int4* chunks = nullptr;          // [nchunks]: the spans in blocks of at most 64 rows: row, rows, adapter
  int32_t* chunk_ptr = nullptr;    // [n_adapters + 1]: where each adapter's blocks start
  std::vector<int32_t> host_chunk_ptr;
  int32_t* empty = nullptr;        // [nempty]: the adapters without rows
  int32_t* used = nullptr;         // [nused]: the adapters with rows, ascending
  int4* pieces = nullptr;          // [npieces]: the segments in pieces of at most 8 rows (up to kRowsMost rows): row, rows, adapter
  cudaStream_t built_on = nullptr;
  cudaEvent_t built = nullptr;     // the arrays are on the device
  bool settled = false;            // `built` has been seen complete
  bool shared = false;             // used on another stream than built_on
};

// The adapter of row t, or -1: the last of the segments meeting its 128 rows that begins at or before it.
__device__ __forceinline__ int adapter_of_row(const int2* tiles, const int4* segs, int64_t t) {
  const int2 tile = __ldg(tiles + t / 128);
  int lo = tile.x, n = tile.y;
  if (!n) return -1;
  while (n > 1) {
    const int h = n / 2;
    if (__ldg(&segs[lo + h].x) <= t) lo += h, n -= h;
    else n = h;
  }
  const int4 s = __ldg(segs + lo);
  return t >= s.x && t < s.y ? s.z : -1;
}

// u and g pass from kernel to kernel as 16-bit parts whose sum is the f32 value,
// R = adapter_rank_rows(rank) columns per part:
//   Q  bf16 [rows, 3·R]  the value, its remainder and the remainder of that: 8 bits each make f32's 24, over f32's range.
//                        Read beside the projection (lc_gemm.cu, lc_adapters_rows.cu) and, in bf16, by the outer sums.
//   H  f16 [rows, 4·R]   parts in units of 2^19, 2^8, 2^-3 and 2^-14, read by the outer sums of f16: their other operand
//                        is f16, which an MMA cannot mix with bf16. Each part takes 11 bits of what the ones before left:
//                        exact to 2^-39 up to 3.4e10 (beyond: inf), so neither a loss gradient of 1e-6 a row nor one
//                        scaled by 2^16 loses bits that f32 keeps. Two f16 parts without units held no more than 2^-25,
//                        1e-2 of the gradients for a dy of 3e-6 over 4096 rows. The first two parts are left at zero
//                        where they would be subnormal: the tensor cores align a subnormal operand's products by the
//                        smallest normal exponent, and the running sum loses the bits below that window (997 rows, dA:
//                        0.39 % of the results a neighbour of the exact value rounded, against 0.04 %). Where the third
//                        is subnormal (below 2^-17) that costs 2^-41 a step and its bits are worth more.
constexpr int kQParts = 3, kHParts = 4;
inline int adapter_rank_rows(int rank) { return rank <= 32 ? (rank + 15) / 16 * 16 : (rank + 63) / 64 * 64; }

__device__ __forceinline__ void split_bf16(float v, __nv_bfloat16 (&q)[kQParts]) {
  q[0] = __float2bfloat16_rn(v);
  q[1] = q[2] = __float2bfloat16_rn(0.f);
  if (!isfinite(v)) return;  // the value itself: its remainder would be NaN
  if (!isfinite(__bfloat162float(q[0]))) q[0] = __float2bfloat16_rn(copysignf(0x1.fep127f, v));
  const float r = v - __bfloat162float(q[0]);
  q[1] = __float2bfloat16_rn(r);
  q[2] = __float2bfloat16_rn(r - __bfloat162float(q[1]));
}
__device__ __forceinline__ void split_f16(float v, __half (&h)[kHParts]) {
  const bool in = fabsf(v) < 0x1.ffcp34f;
  float r = in ? v : 0.f;
  const float unit[kHParts] = {0x1p19f, 0x1p8f, 0x1p-3f, 0x1p-14f}, per[kHParts] = {0x1p-19f, 0x1p-8f, 0x1p3f, 0x1p14f};
#pragma unroll
  for (int i = 0; i < kHParts; i++) {
    h[i] = __float2half_rn(i >= 2 || fabsf(r) >= unit[i] * 0x1p-14f ? r * per[i] : 0.f);
    r -= __half2float(h[i]) * unit[i];
  }
  if (!in) h[0] = __float2half_rn(isnan(v) ? v : copysignf(INFINITY, v));
}

// The rows of an f16 bank [n, rank, cols] that a batch uses, as bf16 values and
// remainders [used adapters, 2·R, ld] with zeros from the rank on: the 11 bits
// of an f16 as two bf16, which the tensor cores multiply with the bf16 parts of
// u (lc_gemm.cu). Eight values of a row per step.
struct BankSplit {
  const uint16_t* src = nullptr;
  uint16_t* dst = nullptr;
  const int32_t* used = nullptr;
  int64_t cols = 0, ld = 0, steps = 0;
  int rank = 0, R = 0, vec = 0;  // vec: the source rows are 16-byte aligned
};
// Values c .. c + 7 of a row of `cols`, zeros from its end on.
__device__ __forceinline__ uint4 row_values8(const uint16_t* row, int64_t cols, int64_t c, bool vec) {
  if (vec) return __ldg((const uint4*)(row + c));
  alignas(16) uint16_t v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) v[e] = c + e < cols ? row[c + e] : (uint16_t)0;
  return *(const uint4*)v;
}
__device__ __forceinline__ void split_bank_step(const BankSplit& b, int64_t i) {
  const int64_t vecs = b.ld / 8, row = i / vecs, c = (i % vecs) * 8, slot = row / b.R, r = row % b.R;
  const uint4 v = r < b.rank ? row_values8(b.src + (__ldg(b.used + slot) * (int64_t)b.rank + r) * b.cols, b.cols, c, b.vec) : make_uint4(0u, 0u, 0u, 0u);
  alignas(16) __nv_bfloat16 high[8], low[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const float f = __half2float(((const __half*)&v)[e]);
    high[e] = __float2bfloat16_rn(f);
    low[e] = __float2bfloat16_rn(isfinite(f) ? f - __bfloat162float(high[e]) : 0.f);
  }
  uint4* d = (uint4*)(b.dst + (slot * 2 * b.R + r) * b.ld + c);
  *d = *(const uint4*)high;
  d[b.R * vecs] = *(const uint4*)low;
}

// s_a·P_a·X[t] as Q and H (each may be null) for X [rows, C] and P [n, rank, C] (row strides ld, ldp: multiples of 8;
// 16-byte aligned).
struct AdapterShrink {
  const void *X = nullptr, *P = nullptr;
  int64_t C = 0, ld = 0, ldp = 0;
  int n = 0, rank = 0;
  const float* scales = nullptr;
  __nv_bfloat16* Q = nullptr;
  __half* H = nullptr;
};
// dP[a] = Σ_{t in a} q[t] ⊗ X[t], [n, rank, C] dense; `parts` holds q as Q (bf16) or H (f16).
struct AdapterOuter {
  const void *X = nullptr, *parts = nullptr;
  int64_t C = 0, ld = 0;
  int rank = 0;
  void* dP = nullptr;
};
namespace lc {
// One or two products over the same rows, ranks and scales.
void adapter_shrink_tc(const AdapterShrink* c, int njobs, const AdapterPlan& p, int dtype, cudaStream_t st);
size_t adapter_part_bytes(const AdapterOuter* c, int njobs, const AdapterPlan& p);  // f32 partial sums of adapter_outer_tc
void adapter_outer_tc(const AdapterOuter* c, int njobs, void* part, const AdapterPlan& p, int dtype, cudaStream_t st);
// The forms for few rows (lc_adapters_rows.cu) fit up to so many
// multiplications. Measured (bf16, rank 16, 768 columns; dot
// products against tensor cores, one request / requests of 8 rows): shrink
// 25 M 6.0 / 8.1 us against 8.3 / 16.4, 50 M 10.1 / 13.7 against 8.5 / 16.2;
// linear 28 M 7.3 us against 9.4 / 9.7, 57 M 13.3 against 9.5 / 10.4. Twice
// as many where requests are short: 1000 rows in 200 requests, 1024 columns,
// rank 40 (66 M each) take 17 and 14 us against 25 and 44.
constexpr int kRowsMost = 16384;
constexpr int64_t kRowsShrinkMost = 3 << 24, kRowsLinearMost = 1 << 25;
bool adapter_shrink_rows_fit(const AdapterShrink* c, int njobs, const AdapterPlan& p);
// `split` (steps may be 0) rides along in blocks of its own.
void adapter_shrink_rows(const AdapterShrink* c, int njobs, const BankSplit& split, const AdapterPlan& p, int dtype, cudaStream_t st);
bool adapter_linear_rows_fit(int64_t M, int64_t N, int64_t K, const AdapterPlan& p);
// The forward product for a call that fits; c.share.bank [n, rank, ld] is in `dtype` here.
void adapter_linear_rows(const GemmAdaptedCall& c, const AdapterPlan& p, int rank, int dtype, cudaStream_t st);
}  // namespace lc

void lc_adapters_destroy();
