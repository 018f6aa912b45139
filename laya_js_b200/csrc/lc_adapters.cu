// Low-rank adapters of many requests beside a shared projection, and their
// gradients (include/laya_cuda_adapters.h).
//
// Three products make both directions, because the banks keep their long axis
// contiguous (A [n, r, K], B [n, r, N]) and enter symmetrically:
//   shrink  Q[t, :] = s_a · P_a · X[t]             u (X = x, P = A), g (X = dy, P = B)
//   expand  Y[t, :] = W-product of X[t] + P_aᵀ·Q[t] y (P = B), dx (P = A, W read transposed)
//   outer   dP_a    = Σ_{t in a} Q[t] ⊗ X[t]       dA (Q = g, X = x), dB (Q = u, X = dy)
//
// f16 and bf16 run on the tensor cores (lc_adapters_tc.cu, gemm_adapted in
// lc_gemm.cu) or, with few rows, as dot products (lc_adapters_rows.cu). Both
// read 16-byte aligned rows: operands with other widths or addresses are
// copied into padded rows first. The kernels of this file serve f32: one
// thread block per tile, f32 sums in registers, Q in f32.
#include "lc_adapters.h"
#include "lc_api.h"
#include "lc_gemm.h"
#include "laya_cuda_adapters.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <unordered_set>
#include <vector>

namespace {
using namespace lc;

// ------------------------------------------------------------- the plan

std::unordered_set<AdapterPlan*>& plans() {
  static std::unordered_set<AdapterPlan*> s;
  return s;
}

AdapterPlan* check_plan(uint64_t h) {
  AdapterPlan* p = reinterpret_cast<AdapterPlan*>(h);
  LC_CHECK(h && plans().count(p), "adapters: invalid or freed plan handle");
  return p;
}

// The plan's arrays are written once, by the copy that builds it: a use on
// another stream waits for that copy.
void plan_enter(AdapterPlan* p) {
  cudaStream_t st = stream();
  // (cudaStreamPerThread names another stream in every thread)
  if (st == p->built_on && st != cudaStreamPerThread) return;
  p->shared = true;
  if (p->settled || (p->settled = cudaEventQuery(p->built) == cudaSuccess)) return;
  cudaGetLastError();
  // a capturing stream cannot wait for an event recorded outside the capture
  if (capturing()) CUDA_OK(cudaEventSynchronize(p->built));
  else CUDA_OK(cudaStreamWaitEvent(st, p->built, 0));
}

void plan_release(AdapterPlan* p) {
  if (p->shared && !capturing()) cudaDeviceSynchronize();  // the memory is freed in the order of one stream
  if (p->dev) dfree(p->dev);
  if (p->built) cudaEventDestroy(p->built);
  delete p;
}

// ------------------------------------------------------------- f32

// Q[t, j] = s_a · Σ_k X[t, k]·P[a, j, k]; rows without an adapter get zeros.
// A block per row, a warp per rank row j; bound by the reads of P from L2
// (4096 rows of 768, rank 16: 21 us).
__global__ void __launch_bounds__(128) k_shrink_f32(const float* __restrict__ X, const float* __restrict__ P, const float* __restrict__ scales,
                                                    const int2* __restrict__ tiles, const int4* __restrict__ segs, float* __restrict__ Q, int C,
                                                    int r) {
  pdl_trigger();
  pdl_wait();
  const int64_t t = blockIdx.x;
  const int a = adapter_of_row(tiles, segs, t), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float s = a >= 0 ? (scales ? scales[a] : 1.f) : 0.f;
  const float* x = X + t * C;
  for (int j = warp; j < r; j += 4) {
    float acc = 0.f;
    if (a >= 0) {
      const float* p = P + ((int64_t)a * r + j) * C;
      for (int k = lane; k < C; k += 32) acc = fmaf(x[k], p[k], acc);
#pragma unroll
      for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    }
    if (lane == 0) Q[t * r + j] = a >= 0 ? s * acc : 0.f;
  }
}

// Y[m, n] = Σ_k X[m, k]·W(n, k) (+ bias[n]) + Σ_j Q[m, j]·P[a(m), j, n], with
// W(n, k) = W[n·swn + k·swk]. 64 x 64 tiles, 4 x 4 outputs per thread; bound by
// the FMA pipe and the shared-memory loads that feed it (4096 rows, 768 -> 768:
// 217 us, 22 TFLOP/s; the contract's f32 linear takes 389).
__global__ void __launch_bounds__(256) k_expand_f32(const float* __restrict__ X, const float* __restrict__ W, int64_t swn, int64_t swk,
                                                    const char* bias, int bias_dtype, const float* __restrict__ Q,
                                                    const float* __restrict__ P, const int2* __restrict__ tiles, const int4* __restrict__ segs,
                                                    float* __restrict__ Y,
                                                    int64_t M, int N, int K, int r) {
  pdl_trigger();
  pdl_wait();
  __shared__ float xs[16][64 + 4], ws[16][64 + 4];
  const int64_t m0 = (int64_t)blockIdx.x * 64;
  const int n0 = blockIdx.y * 64, tid = threadIdx.x, tm = (tid >> 4) * 4, tn = (tid & 15) * 4;
  float acc[4][4] = {};
  if (W)
    for (int k0 = 0; k0 < K; k0 += 16) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int e = tid + 256 * i;
        {
          const int m = e >> 4, k = e & 15;
          xs[k][m] = (m0 + m < M && k0 + k < K) ? X[(m0 + m) * K + k0 + k] : 0.f;
        }
        // the fast index of the load follows W's contiguous axis
        const int n = swk == 1 ? e >> 4 : e & 63, k = swk == 1 ? e & 15 : e >> 6;
        ws[k][n] = (n0 + n < N && k0 + k < K) ? W[(n0 + n) * swn + (k0 + k) * swk] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; k++) {
        const float4 xv = *(const float4*)&xs[k][tm], wv = *(const float4*)&ws[k][tn];
        const float xa[4] = {xv.x, xv.y, xv.z, xv.w}, wa[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[i][j] = fmaf(xa[i], wa[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t m = m0 + tm + i;
    if (m >= M) break;
    const int a = adapter_of_row(tiles, segs, m);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int n = n0 + tn + j;
      if (n >= N) break;
      float v = acc[i][j];
      if (bias) v += ld_as<float>(bias, bias_dtype, n);
      if (a >= 0) {
        const float* p = P + (int64_t)a * r * N + n;
        const float* q = Q + m * r;
        float d = 0.f;
        for (int l = 0; l < r; l++) d = fmaf(q[l], p[(int64_t)l * N], d);
        v += d;
      }
      Y[m * N + n] = v;
    }
  }
}

// dP[a, j, c] = Σ_{t in a} Q[t, j]·X[t, c]: a block per adapter, 8 rank rows
// and 128 columns; rows in order, in groups of 64 so that a long sum loses no
// more than a short one. Bound by the latency of a block's rows, which follow
// one another (4096 rows of 768, 8 adapters of rank 16: 66 us, eight rows'
// loads at a time; one at a time 124).
__global__ void __launch_bounds__(128) k_outer_f32(const float* __restrict__ Q, const float* __restrict__ X, const int2* __restrict__ spans,
                                                   const int32_t* __restrict__ span_ptr, float* __restrict__ dP, int C, int r) {
  pdl_trigger();
  pdl_wait();
  const int a = blockIdx.z, j0 = blockIdx.y * 8, c = blockIdx.x * 128 + threadIdx.x, cc = min(c, C - 1);
  const int nj = min(8, r - j0);
  float acc[8] = {};
  for (int s = span_ptr[a]; s < span_ptr[a + 1]; s++) {
    const int2 rows = spans[s];
    for (int64_t t0 = rows.x; t0 < rows.y; t0 += 64) {
      const int64_t t1 = min(t0 + 64, (int64_t)rows.y);
      float part[8] = {};
#pragma unroll 8
      for (int64_t t = t0; t < t1; t++) {
        const float x = X[t * C + cc];
        const float* q = Q + t * r + j0;
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (j < nj) part[j] = fmaf(q[j], x, part[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) acc[j] += part[j];
    }
  }
  if (c < C)
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < nj) dP[((int64_t)a * r + j0 + j) * C + c] = acc[j];
}

// ------------------------------------------------------------- operands

// Scratch kept from call to call (padded operands, Q, partial sums): an
// allocation and its release cost 1.2 us each call, a tenth of a small one.
// It belongs to the stream of its first use (the library's own or CUDA's legacy
// default one, which nobody can destroy), whose order separates one call's
// contents from the next; calls on other streams, in captures and beyond
// kMost allocate theirs. It grows to what the calls before have asked for.
struct Workspace {
  static constexpr size_t kMost = (size_t)32 << 20;
  char* p = nullptr;
  size_t bytes = 0, want = 0;
  cudaStream_t st = nullptr;
  bool usable() {
    if (capturing() || !want || !permanent_stream() || (p && st != stream())) return false;
    if (want > bytes) {
      if (p) dfree(p);
      p = nullptr;
      bytes = 0;
      const size_t n = want;
      want = 0;  // (set again below: a failed allocation is not tried at every call)
      p = (char*)dmalloc(n);
      st = stream();
      want = bytes = n;
    }
    return p != nullptr;
  }
};
Workspace& workspace() {
  static Workspace w;
  return w;
}

struct Held {  // tensors and scratch of one call, released when it returns or throws
  std::vector<LcTensor*> ts;
  std::vector<void*> mem;
  const bool kept = workspace().usable();
  size_t used = 0, asked = 0;  // of the workspace; in all
  ~Held() {
    for (auto* t : ts) release(t);
    for (void* p : mem) dfree(p);
    Workspace& w = workspace();
    if (asked <= Workspace::kMost && asked > w.want && !capturing()) w.want = (asked + 65535) / 65536 * 65536;
  }
  LcTensor* dense(LcTensor* t) {
    LcTensor* c = contiguous(t);
    if (c != t) ts.push_back(c);
    return c;
  }
  LcTensor* made(LcTensor* t) {
    ts.push_back(t);
    return t;
  }
  void* scratch(size_t bytes) {
    bytes = (bytes + 255) / 256 * 256;
    asked += bytes;
    if (kept && used + bytes <= workspace().bytes) {
      used += bytes;
      return workspace().p + used - bytes;
    }
    mem.push_back(nullptr);
    return mem.back() = dmalloc(bytes);
  }
  LcTensor* keep(LcTensor* t) {  // handed to the caller: no longer released here
    ts.erase(std::find(ts.begin(), ts.end(), t));
    return t;
  }
};

struct Operands {
  AdapterPlan* plan = nullptr;
  LcTensor *x = nullptr, *dy = nullptr, *w = nullptr, *bias = nullptr, *a = nullptr, *b = nullptr, *scales = nullptr;
  int64_t T = 0, K = 0, N = 0;
  int r = 0, n = 0, dtype = 0;
  const float* scale_ptr() const { return scales ? (const float*)scales->data() : nullptr; }
};

Operands operands(const char* op, lc_tensor xh, lc_tensor dyh, lc_tensor wh, lc_tensor biash, lc_tensor ah, lc_tensor bh, lc_tensor sh,
                  uint64_t planh, Held& held) {
  const std::string name(op);
  Operands o;
  o.plan = check_plan(planh);
  LcTensor* x = check(xh, op);
  LcTensor* a = check(ah, op);
  LcTensor* b = check(bh, op);
  LcTensor* w = wh ? check(wh, op) : nullptr;
  LcTensor* dy = dyh ? check(dyh, op) : nullptr;
  LcTensor* bias = biash ? check(biash, op) : nullptr;
  LcTensor* s = sh ? check(sh, op) : nullptr;
  o.dtype = x->dtype;
  LC_CHECK(o.dtype == LC_F32 || is_half(o.dtype), name + ": x must be f32, f16 or bf16, got " + dtype_name(o.dtype));
  LC_CHECK(x->ndim >= 1, name + ": x [..., in] expected");
  LC_CHECK(a->ndim == 3 && b->ndim == 3, name + ": a [n, r, in] and b [n, r, out] expected");
  for (LcTensor* t : {a, b, w, dy})
    if (t) LC_CHECK(t->dtype == o.dtype, name + ": x, w, a, b (and dy) must share a dtype, got " + dtype_name(o.dtype) + " and " + dtype_name(t->dtype));
  o.K = x->shape[x->ndim - 1];
  o.N = b->shape[2];
  const int64_t rows = o.K ? x->numel() / o.K : 0;
  LC_CHECK(o.K >= 1 && o.N >= 1, name + ": in and out must be at least 1");
  LC_CHECK(o.K <= INT32_MAX / 8 && o.N <= INT32_MAX / 8, name + ": in or out is too large");
  LC_CHECK(a->shape[2] == o.K, name + ": x " + shape_str(x->dims()) + " vs a " + shape_str(a->dims()));
  LC_CHECK(a->shape[0] == b->shape[0] && a->shape[1] == b->shape[1], name + ": a " + shape_str(a->dims()) + " vs b " + shape_str(b->dims()));
  LC_CHECK(a->shape[0] == o.plan->n_adapters,
           name + ": the plan was made for " + std::to_string(o.plan->n_adapters) + " adapters, a " + shape_str(a->dims()));
  LC_CHECK(a->shape[1] >= 1 && a->shape[1] <= kAdapterMaxRank, name + ": rank must be 1 to " + std::to_string(kAdapterMaxRank));
  LC_CHECK(rows == o.plan->rows, name + ": x has " + std::to_string(rows) + " rows, the plan " + std::to_string(o.plan->rows));
  if (w) LC_CHECK(w->ndim == 2 && w->shape[0] == o.N && w->shape[1] == o.K,
                  name + ": w " + shape_str(w->dims()) + ", expected [" + std::to_string(o.N) + "," + std::to_string(o.K) + "]");
  if (bias) LC_CHECK(bias->numel() == o.N && (bias->dtype == LC_F32 || is_half(bias->dtype)), name + ": bias must hold out f32, f16 or bf16 values");
  if (s) LC_CHECK(s->dtype == LC_F32 && s->ndim == 1 && s->shape[0] == a->shape[0], name + ": scales must be f32 [n]");
  if (dy) {
    std::vector<int64_t> want = x->dims();
    want.back() = o.N;
    LC_CHECK(dy->dims() == want, name + ": dy " + shape_str(dy->dims()) + ", expected " + shape_str(want));
  }
  o.T = rows;
  o.r = (int)a->shape[1];
  o.n = (int)a->shape[0];
  o.x = held.dense(x);
  o.a = held.dense(a);
  o.b = held.dense(b);
  if (w) o.w = held.dense(w);
  if (dy) o.dy = held.dense(dy);
  if (bias) o.bias = held.dense(bias);
  if (s) o.scales = held.dense(s);
  plan_enter(o.plan);
  return o;
}

// ------------------------------------------------------------- f32 forms

void shrink_f32(const Operands& o, const LcTensor* X, const LcTensor* P, int64_t C, float* Q) {
  launch_chain(k_shrink_f32, dim3((unsigned)o.T), dim3(128), 0, stream(), (const float*)X->data(), (const float*)P->data(), o.scale_ptr(),
               (const int2*)o.plan->tiles, (const int4*)o.plan->segs, Q, (int)C, o.r);
  LC_LAUNCHED(1);
}

// y (transposed = false) or dx (transposed = true)
void expand_f32(const Operands& o, const LcTensor* X, const LcTensor* P, const float* Q, bool transposed, LcTensor* Y) {
  const int64_t in = transposed ? o.N : o.K, out = transposed ? o.K : o.N;
  const LcTensor* bias = transposed ? nullptr : o.bias;
  dim3 grid((unsigned)((o.T + 63) / 64), (unsigned)((out + 63) / 64));
  LC_CHECK(grid.y <= 65535, "adapters: too many output columns");
  launch_chain(k_expand_f32, grid, dim3(256), 0, stream(), (const float*)X->data(), o.w ? (const float*)o.w->data() : (const float*)nullptr,
               transposed ? (int64_t)1 : o.K, transposed ? o.K : (int64_t)1, bias ? (const char*)bias->data() : (const char*)nullptr,
               bias ? bias->dtype : 0, Q, (const float*)P->data(), (const int2*)o.plan->tiles, (const int4*)o.plan->segs, (float*)Y->data(), o.T, (int)out,
               (int)in, o.r);
  LC_LAUNCHED(1);
}

void outer_f32(const Operands& o, const float* Q, const LcTensor* X, int64_t C, LcTensor* dP) {
  dim3 grid((unsigned)((C + 127) / 128), (unsigned)((o.r + 7) / 8), (unsigned)o.n);
  LC_CHECK(grid.z <= 65535, "adapters: more than 65535 adapters");
  launch_chain(k_outer_f32, grid, dim3(128), 0, stream(), Q, (const float*)X->data(), (const int2*)o.plan->spans,
               (const int32_t*)o.plan->span_ptr, (float*)dP->data(), (int)C, o.r);
  LC_LAUNCHED(1);
}

// ------------------------------------------------------------- 16-bit forms

// A row-major matrix (or a stack of them) whose rows TMA can read.
struct Rows {
  const void* p = nullptr;
  int64_t ld = 0;
};

// Copies rows of `cols` values into rows of `ld` (a multiple of 8), zeros after
// them, eight values per thread step, up to five matrices a launch, the steps
// of all of them in one range, and after them those of a bank's split. Bound by
// the latency of the 2-byte loads (1537 x 1001, 777 x 1001 and two banks: 3.9
// us; matrix after matrix 4.4).
struct PadJob {
  const uint16_t* src;
  uint16_t* dst;
  int64_t first, cols, ld;  // first: steps of the matrices before it
};
struct PadJobs {
  int n;
  int64_t total;
  PadJob j[5];
  BankSplit split;
};
__global__ void __launch_bounds__(256) k_pad_rows(const __grid_constant__ PadJobs jobs) {
  pdl_trigger();
  pdl_wait();
  LC_GRID_STRIDE(g, jobs.total + jobs.split.steps) {
    if (g >= jobs.total) {
      split_bank_step(jobs.split, g - jobs.total);
      continue;
    }
    int k = jobs.n - 1;
    while (g < jobs.j[k].first) k--;
    const PadJob& j = jobs.j[k];
    const int64_t i = g - j.first, vecs = j.ld / 8, row = i / vecs, c = (i % vecs) * 8;
    *(uint4*)(j.dst + row * j.ld + c) = row_values8(j.src + row * j.cols, j.cols, c, false);
  }
}

struct Padder {
  Held& held;
  PadJobs jobs{};
  BankSplit split{};
  static bool aligned(const LcTensor* t, int64_t cols) { return cols % 8 == 0 && ((uintptr_t)t->data() & 15) == 0; }
  Rows of(const LcTensor* t, int64_t rows, int64_t cols) {
    if (!t) return {};
    if (aligned(t, cols)) return {t->data(), cols};
    const int64_t ld = (cols + 7) / 8 * 8;
    void* d = held.scratch((size_t)(rows * ld) * 2);
    jobs.j[jobs.n++] = {(const uint16_t*)t->data(), (uint16_t*)d, jobs.total, cols, ld};
    jobs.total += rows * ld / 8;
    return {d, ld};
  }
  // The bank beside a projection on the tensor cores: bf16 rows, or those of an f16 bank's used adapters in two parts.
  Rows share(const LcTensor* bank, const AdapterPlan& p, int rank, int64_t cols) {
    if (bank->dtype == LC_BF16) return of(bank, bank->shape[0] * rank, cols);
    split.ld = (cols + 7) / 8 * 8;
    split.cols = cols;
    split.rank = rank;
    split.R = adapter_rank_rows(rank);
    split.vec = aligned(bank, cols);
    split.used = p.used;
    split.src = (const uint16_t*)bank->data();
    const int64_t rows = (int64_t)p.nused * split.R;
    split.dst = (uint16_t*)held.scratch((size_t)(2 * rows * split.ld) * 2);
    split.steps = rows * split.ld / 8;
    return {split.dst, split.ld};
  }
  // Launches the copies, with the split among them unless it may ride with the shrink and there is nothing else to do
  // (128 rows of f16 through 768 -> 2304: 2.2 us for a launch of its own). True when a kernel was launched: the next one
  // may start while it runs, and waits for it.
  bool run(bool split_may_ride) {
    if (!split_may_ride || jobs.total) std::swap(jobs.split, split);
    const int64_t steps = jobs.total + jobs.split.steps;
    if (!steps) return false;
    launch_chain(k_pad_rows, dim3(blocks_for(steps, 256)), dim3(256), 0, stream(), jobs);
    LC_LAUNCHED(1);
    return true;
  }
};

// The kernels after the shrink start while it runs (programmatic dependent
// launch). It releases them after its own dependency wait, so what ran before
// this operator is complete by then, and each waits for its predecessor before
// it reads what that wrote and before it ends.
struct Chained {
  std::unique_ptr<PdlScope> scope;
  explicit Chained(const Operands& o) {
    if (o.plan->nsegs) scope = std::make_unique<PdlScope>();
  }
};

// Room for u or g as Q and as H, and the product that fills them.
size_t parts_bytes(const Operands& o, int parts) { return ((size_t)o.T * parts * adapter_rank_rows(o.r) * 2 + 255) / 256 * 256; }
AdapterShrink shrink_job(const Operands& o, const Rows& X, const Rows& P, int64_t C, void* Q, void* H) {
  AdapterShrink c;
  c.X = X.p;
  c.P = P.p;
  c.C = C;
  c.ld = X.ld;
  c.ldp = P.ld;
  c.n = o.n;
  c.rank = o.r;
  c.scales = o.scale_ptr();
  c.Q = (__nv_bfloat16*)Q;
  c.H = (__half*)H;
  return c;
}

// The copies and the narrow products.
void shrink(const AdapterShrink* c, int njobs, const Operands& o, Padder& pad) {
  const bool few = adapter_shrink_rows_fit(c, njobs, *o.plan);
  std::unique_ptr<PdlScope> chained = pad.run(few) ? std::make_unique<PdlScope>() : nullptr;
  if (few) adapter_shrink_rows(c, njobs, pad.split, *o.plan, o.dtype, stream());
  else adapter_shrink_tc(c, njobs, *o.plan, o.dtype, stream());
}

// y, or dx (transposed). `few`: the dot-product form, whose bank is in the operands' type; otherwise `bank` is Padder::share's.
void expand_16(const Operands& o, const Rows& X, const Rows& W, const Rows& bank, const void* Q, bool transposed, bool few, LcTensor* Y) {
  GemmAdaptedCall c;
  c.x = X.p;
  c.M = o.T;
  c.K = transposed ? o.N : o.K;
  c.ldx = X.ld;
  c.w = W.p;
  c.ldw = W.ld;
  c.N = transposed ? o.K : o.N;
  c.transposed = transposed;
  if (o.bias && !transposed) {
    c.bias = o.bias->data();
    c.bias_dtype = o.bias->dtype;
  }
  c.y = Y->data();
  c.ldy = c.N;
  c.share.u = Q;
  c.share.R = adapter_rank_rows(o.r);
  c.share.bank = bank.p;
  c.share.ld = bank.ld;
  c.share.parts = o.dtype == LC_F16 ? 2 : 1;
  c.share.n = o.dtype == LC_F16 ? o.plan->nused : o.n;
  c.share.rows = o.dtype == LC_F16 ? 2 * c.share.R : o.r;
  c.share.nsegs = o.plan->nsegs;
  c.share.segs = o.plan->segs;
  c.share.tiles = o.plan->tiles;
  c.after_share = o.plan->nsegs > 0;
  if (few) adapter_linear_rows(c, *o.plan, o.r, o.dtype, stream());
  else gemm_adapted(c, o.dtype, stream());
}

void linear(const Operands& o, LcTensor* y, Held& held) {
  if (!o.T) return;
  if (o.dtype == LC_F32) {
    float* u = (float*)held.scratch((size_t)o.T * o.r * 4);
    shrink_f32(o, o.x, o.a, o.K, u);
    expand_f32(o, o.x, o.b, u, false, y);
    return;
  }
  const bool few = adapter_linear_rows_fit(o.T, o.N, o.K, *o.plan);
  Padder pad{held};
  const Rows x = pad.of(o.x, o.T, o.K), w = pad.of(o.w, o.N, o.K), a = pad.of(o.a, (int64_t)o.n * o.r, o.K),
             b = few ? pad.of(o.b, (int64_t)o.n * o.r, o.N) : pad.share(o.b, *o.plan, o.r, o.N);
  const AdapterShrink u = shrink_job(o, x, a, o.K, held.scratch(parts_bytes(o, kQParts)), nullptr);
  shrink(&u, 1, o, pad);
  const Chained chained(o);
  expand_16(o, x, w, b, u.Q, false, few, y);
}

void gradients(const Operands& o, LcTensor* dx, LcTensor* da, LcTensor* db, Held& held) {
  if (!o.plan->nsegs) {  // no row has an adapter
    for (LcTensor* t : {da, db})
      if (t && t->numel()) CUDA_OK(cudaMemsetAsync(t->data(), 0, t->numel() * dtype_size(o.dtype), stream()));
    da = db = nullptr;
    if (!o.T) return;
  }
  if (o.dtype == LC_F32) {
    float* q = (float*)held.scratch((size_t)o.T * o.r * 4);
    if (dx || da) {
      shrink_f32(o, o.dy, o.b, o.N, q);
      if (dx) expand_f32(o, o.dy, o.a, q, true, dx);
      if (da) outer_f32(o, q, o.x, o.K, da);
    }
    if (db) {
      shrink_f32(o, o.x, o.a, o.K, q);
      outer_f32(o, q, o.dy, o.N, db);
    }
    return;
  }
  const bool f16 = o.dtype == LC_F16;
  Padder pad{held};
  const Rows dy = pad.of(o.dy, o.T, o.N), x = da || db ? pad.of(o.x, o.T, o.K) : Rows{}, w = dx ? pad.of(o.w, o.N, o.K) : Rows{},
             a = db || (dx && !f16) ? pad.of(o.a, (int64_t)o.n * o.r, o.K) : Rows{},
             b = dx || da ? pad.of(o.b, (int64_t)o.n * o.r, o.N) : Rows{}, bank = dx && f16 ? pad.share(o.a, *o.plan, o.r, o.K) : a;
  AdapterOuter out[2];
  int no = 0;
  auto job = [&](const Rows& X, int64_t C, LcTensor* dP) {
    AdapterOuter& c = out[no++];
    c.X = X.p;
    c.C = C;
    c.ld = X.ld;
    c.rank = o.r;
    c.dP = dP->data();
  };
  if (db) job(dy, o.N, db);
  if (da) job(x, o.K, da);
  // beside the projection g is read as Q; the outer sums read u and g in the type of the rows they meet
  const size_t q_bytes = parts_bytes(o, kQParts), h_bytes = parts_bytes(o, kHParts);
  const bool gq = dx || (da && !f16), gh = da && f16;
  size_t at = 0;
  auto place = [&](bool want, size_t bytes) {
    const size_t here = at;
    if (want) at += bytes;
    return here;
  };
  const size_t u_at = place(db != nullptr, f16 ? h_bytes : q_bytes), gq_at = place(gq, q_bytes), gh_at = place(gh, h_bytes);
  if (!at) return;
  char* scratch = (char*)held.scratch(at + (no ? adapter_part_bytes(out, no, *o.plan) : 0));
  AdapterShrink q[2];
  int nq = 0;
  if (db) {
    q[nq++] = shrink_job(o, x, a, o.K, f16 ? nullptr : scratch + u_at, f16 ? scratch + u_at : nullptr);
    out[0].parts = scratch + u_at;
  }
  if (dx || da) q[nq++] = shrink_job(o, dy, b, o.N, gq ? scratch + gq_at : nullptr, gh ? scratch + gh_at : nullptr);
  if (da) out[no - 1].parts = scratch + (f16 ? gh_at : gq_at);
  shrink(q, nq, o, pad);
  const Chained chained(o);
  if (no) adapter_outer_tc(out, no, scratch + at, *o.plan, o.dtype, stream());
  if (dx) expand_16(o, dy, w, bank, scratch + gq_at, true, false, dx);
}

}  // namespace

void lc_adapters_destroy() {
  for (auto* p : plans()) plan_release(p);
  plans().clear();
  if (workspace().p) cudaFree(workspace().p);  // waits for its uses, on whichever stream
  workspace() = Workspace();
}

extern "C" {

int lc_adapter_plan_create(uint64_t* out, const int32_t* cu_rows, const int32_t* adapters, int nseg, int n_adapters) {
  LC_API_BEGIN
  cudaStream_t st = stream();
  LC_CHECK(st, "liblaya_cuda: lc_init(device) was not called");
  LC_CHECK(nseg >= 0 && cu_rows && (adapters || !nseg), "adapter plan: cu_rows and adapters are required");
  LC_CHECK(n_adapters >= 0, "adapter plan: n_adapters must be >= 0");
  LC_CHECK(!capturing(), "adapter plan: cannot be created while capturing");
  LC_CHECK(cu_rows[0] == 0, "adapter plan: cu_rows must start at 0");
  for (int i = 0; i < nseg; i++) {
    LC_CHECK(cu_rows[i + 1] >= cu_rows[i], "adapter plan: cu_rows must not decrease (request " + std::to_string(i) + ")");
    LC_CHECK(adapters[i] >= -1 && adapters[i] < n_adapters,
             "adapter plan: request " + std::to_string(i) + " uses adapter " + std::to_string(adapters[i]) + " of " + std::to_string(n_adapters));
  }
  const int T = cu_rows[nseg];
  LC_CHECK(T <= INT32_MAX - 1023, "adapter plan: too many rows");
  // the requests that have rows and an adapter; neighbours with the same adapter become one
  struct Seg { int lo, hi, a; };
  std::vector<Seg> segs;
  for (int i = 0; i < nseg; i++) {
    if (adapters[i] < 0 || cu_rows[i + 1] == cu_rows[i]) continue;
    if (!segs.empty() && segs.back().a == adapters[i] && segs.back().hi == cu_rows[i]) segs.back().hi = cu_rows[i + 1];
    else segs.push_back({cu_rows[i], cu_rows[i + 1], adapters[i]});
  }
  // the arrays of AdapterPlan in one device allocation
  const size_t S = segs.size();
  std::vector<int32_t> span_ptr(n_adapters + 1, 0);
  for (auto& s : segs) span_ptr[s.a + 1]++;
  for (int a = 0; a < n_adapters; a++) span_ptr[a + 1] += span_ptr[a];
  std::vector<int32_t> at(span_ptr.begin(), span_ptr.end() - 1), spans(2 * S);
  for (auto& s : segs) {
    const int k = at[s.a]++;
    spans[2 * k] = s.lo;
    spans[2 * k + 1] = s.hi;
  }
  std::vector<int32_t> seg4, tiles;
  std::vector<int32_t> empty, used, place(n_adapters);
  for (int a = 0; a < n_adapters; a++) {
    std::vector<int32_t>& list = span_ptr[a] == span_ptr[a + 1] ? empty : used;
    place[a] = (int32_t)list.size();
    list.push_back(a);
  }
  for (auto& g : segs) seg4.insert(seg4.end(), {g.lo, g.hi, g.a, place[g.a]});
  for (int64_t m0 = 0, k = 0; m0 < T; m0 += 128) {
    while (k < (int64_t)S && segs[k].hi <= m0) k++;
    int64_t e = k;
    while (e < (int64_t)S && segs[e].lo < m0 + 128) e++;
    tiles.insert(tiles.end(), {(int32_t)k, (int32_t)(e - k)});
  }
  std::vector<int32_t> chunks, chunk_ptr(n_adapters + 1, 0);
  for (int a = 0; a < n_adapters; a++) {
    for (int k = span_ptr[a]; k < span_ptr[a + 1]; k++)
      for (int64_t t = spans[2 * k]; t < spans[2 * k + 1]; t += 64)
        chunks.insert(chunks.end(), {(int32_t)t, (int32_t)std::min<int64_t>(64, spans[2 * k + 1] - t), a, 0});
    chunk_ptr[a + 1] = (int32_t)(chunks.size() / 4);
  }
  std::vector<int32_t> pieces;
  if (T <= kRowsMost)
    for (auto& g : segs)
      for (int t = g.lo; t < g.hi; t += 8) pieces.insert(pieces.end(), {t, std::min(8, g.hi - t), g.a, 0});
  std::vector<int32_t> image;
  auto put = [&](const std::vector<int32_t>& v) {
    const size_t off = image.size();
    image.insert(image.end(), v.begin(), v.end());
    image.resize((image.size() + 63) / 64 * 64);
    return off;
  };
  const size_t o_spans = put(spans), o_ptr = put(span_ptr), o_segs = put(seg4), o_tiles = put(tiles),
               o_chunks = put(chunks), o_chunk_ptr = put(chunk_ptr), o_empty = put(empty),
               o_used = put(used), o_pieces = put(pieces);
  struct Guard {
    AdapterPlan* p;
    ~Guard() { if (p) plan_release(p); }
  } g{new AdapterPlan()};
  AdapterPlan* p = g.p;
  p->rows = T;
  p->n_adapters = n_adapters;
  p->nsegs = (int)S;
  p->nchunks = (int)(chunks.size() / 4);
  p->built_on = st;
  CUDA_OK(cudaEventCreateWithFlags(&p->built, cudaEventDisableTiming));
  p->dev = (int32_t*)dmalloc(image.size() * 4);
  // pageable source: staged when the call returns
  CUDA_OK(cudaMemcpyAsync(p->dev, image.data(), image.size() * 4, cudaMemcpyHostToDevice, st));
  CUDA_OK(cudaEventRecord(p->built, st));
  p->spans = (int2*)(p->dev + o_spans);
  p->span_ptr = p->dev + o_ptr;
  p->segs = (int4*)(p->dev + o_segs);
  p->tiles = (int2*)(p->dev + o_tiles);
  p->chunks = (int4*)(p->dev + o_chunks);
  p->chunk_ptr = p->dev + o_chunk_ptr;
  p->host_chunk_ptr = std::move(chunk_ptr);
  p->empty = p->dev + o_empty;
  p->nempty = (int)empty.size();
  p->used = p->dev + o_used;
  p->nused = (int)used.size();
  p->pieces = (int4*)(p->dev + o_pieces);
  p->npieces = (int)(pieces.size() / 4);
  plans().insert(p);
  g.p = nullptr;
  *out = reinterpret_cast<uint64_t>(p);
  LC_API_END
}

int lc_adapter_plan_free(uint64_t h) {
  LC_API_BEGIN
  AdapterPlan* p = check_plan(h);
  plan_enter(p);
  plans().erase(p);
  plan_release(p);
  LC_API_END
}

int lc_adapter_linear(lc_tensor* out, lc_tensor xh, lc_tensor wh, lc_tensor biash, lc_tensor ah, lc_tensor bh, lc_tensor sh, uint64_t plan) {
  LC_API_BEGIN
  Held held;
  LC_CHECK(out, "adapter_linear: out is required");
  Operands o = operands("adapter_linear", xh, 0, wh, biash, ah, bh, sh, plan, held);
  std::vector<int64_t> shape = check(xh, "adapter_linear")->dims();
  shape.back() = o.N;
  LcTensor* y = held.made(alloc(o.dtype, shape));
  linear(o, y, held);
  *out = handle(held.keep(y));
  LC_API_END
}

int lc_adapter_linear_grad(lc_tensor* dxo, lc_tensor* dao, lc_tensor* dbo, lc_tensor dyh, lc_tensor xh, lc_tensor wh, lc_tensor ah, lc_tensor bh,
                           lc_tensor sh, uint64_t plan) {
  LC_API_BEGIN
  Held held;
  LC_CHECK(dyh, "adapter_linear_grad: dy is required");
  Operands o = operands("adapter_linear_grad", xh, dyh, wh, 0, ah, bh, sh, plan, held);
  LcTensor *dx = nullptr, *da = nullptr, *db = nullptr;
  if (dxo) dx = held.made(alloc(o.dtype, check(xh, "adapter_linear_grad")->dims()));
  if (dao) da = held.made(alloc(o.dtype, o.a->dims()));
  if (dbo) db = held.made(alloc(o.dtype, o.b->dims()));
  gradients(o, dx, da, db, held);
  if (dx) *dxo = handle(held.keep(dx));
  if (da) *dao = handle(held.keep(da));
  if (db) *dbo = handle(held.keep(db));
  LC_API_END
}

}  // extern "C"
