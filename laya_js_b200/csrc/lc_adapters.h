// Internal definitions of the adapter operators (include/laya_cuda_adapters.h).
#pragma once
#include "lc_common.cuh"
#include "lc_gemm.h"

constexpr int kAdapterMaxRank = 256;

// Rows and adapters of one batch on the device (lc_adapter_plan_create).
struct AdapterPlan {
  int rows = 0, n_adapters = 0, nsegs = 0, nchunks = 0, nempty = 0, npieces = 0;
  int32_t* dev = nullptr;          // one allocation behind the arrays below
  int4* segs = nullptr;            // [nsegs]: row ranges with an adapter, ascending: lo, hi, adapter
  int2* tiles = nullptr;           // per 128 rows: the first segment that meets them, and how many do
  int2* spans = nullptr;           // [nsegs]: the row ranges adapter by adapter, ascending within one
  int32_t* span_ptr = nullptr;     // [n_adapters + 1]: where each adapter's spans start
  int4* chunks = nullptr;          // [nchunks]: the spans in blocks of at most 64 rows: row, rows, adapter
  int32_t* chunk_ptr = nullptr;    // [n_adapters + 1]: where each adapter's blocks start
  std::vector<int32_t> host_chunk_ptr;
  int32_t* empty = nullptr;        // [nempty]: the adapters without rows
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

// 16-bit columns of a row of Q (lc_adapters_tc.cu): two parts of the rank
// rounded up to 16, or to 64 above 32, where a part fills whole 128-byte rows.
inline int adapter_u_cols(int rank) { return 2 * (rank <= 32 ? (rank + 15) / 16 * 16 : (rank + 63) / 64 * 64); }

// A value as two 16-bit parts, high part and remainder (Q of lc_adapters_tc.cu).
template <typename T> __device__ __forceinline__ T largest();
template <> __device__ __forceinline__ __half largest<__half>() { return __ushort_as_half(0x7bff); }
template <> __device__ __forceinline__ __nv_bfloat16 largest<__nv_bfloat16>() { return __ushort_as_bfloat16(0x7f7f); }
template <typename T>
__device__ __forceinline__ void split2(float v, T& hi, T& lo) {
  hi = from_f<T>(v);
  float h = to_f<T>(hi);
  if (!isfinite(h)) {
    if (!isfinite(v)) {  // the value itself: its remainder would be NaN
      lo = from_f<T>(0.f);
      return;
    }
    h = copysignf(to_f<T>(largest<T>()), v);
    hi = from_f<T>(h);
  }
  lo = from_f<T>(v - h);
}

// Q[t] = s_a·P_a·X[t] for X [rows, C] and P [n, rank, C] (row strides ld, ldp: multiples of 8; 16-byte aligned).
struct AdapterShrink {
  const void *X = nullptr, *P = nullptr;
  int64_t C = 0, ld = 0, ldp = 0;
  int n = 0, rank = 0;
  const float* scales = nullptr;
  void* Q = nullptr;
};
// dP[a] = Σ_{t in a} Q[t] ⊗ X[t], [n, rank, C] dense.
struct AdapterOuter {
  const void *X = nullptr, *Q = nullptr;
  int64_t C = 0, ld = 0;
  int rank = 0;
  void* dP = nullptr;
};
namespace lc {
// One or two products over the same rows, ranks and scales.
void adapter_shrink_tc(const AdapterShrink* c, int njobs, const AdapterPlan& p, int dtype, cudaStream_t st);
size_t adapter_part_bytes(const AdapterOuter* c, int njobs, const AdapterPlan& p);  // f32 partial sums of adapter_outer_tc
void adapter_outer_tc(const AdapterOuter* c, int njobs, void* part, const AdapterPlan& p, int dtype, cudaStream_t st);
// The forms for few rows (lc_adapters_rows.cu): false, with nothing launched,
// above so many multiplications. Measured (bf16, rank 16, 768 columns; dot
// products against tensor cores, one request / requests of 8 rows): shrink
// 25 M 6.0 / 8.1 us against 8.3 / 16.4, 50 M 10.1 / 13.7 against 8.5 / 16.2;
// linear 28 M 7.3 us against 9.4 / 9.7, 57 M 13.3 against 9.5 / 10.4. Twice
// as many where requests are short: 1000 rows in 200 requests, 1024 columns,
// rank 40 (66 M each) take 17 and 14 us against 25 and 44.
constexpr int kRowsMost = 16384;
constexpr int64_t kRowsShrinkMost = 3 << 24, kRowsLinearMost = 1 << 25;
bool adapter_shrink_rows(const AdapterShrink* c, int njobs, const AdapterPlan& p, int dtype, cudaStream_t st);
bool adapter_linear_rows(const GemmAdaptedCall& c, const AdapterPlan& p, int dtype, cudaStream_t st);
}  // namespace lc

void lc_adapters_destroy();
