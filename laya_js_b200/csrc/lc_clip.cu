// Global-norm gradient clipping over many tensors (lc_clip_grad_norm,
// include/laya_cuda_adapters.h): norm = sqrt(Σ g²), out = g·min(1, max/(norm + 1e-6)).
//
// Every tensor is cut into chunks of kChunk elements; block b takes chunks b,
// b + grid, ... Pass one leaves one f64 partial sum of squares per block, pass
// two adds the partials in a fixed order in every block and scales.
#include "lc_api.h"
#include "laya_cuda_adapters.h"

#include <algorithm>
#include <cmath>
#include <vector>

namespace {
using namespace lc;

constexpr int kChunk = 8192;       // elements per chunk
constexpr int kMaxTensors = 640;   // per launch: the table travels as a kernel parameter (at most 32 KB)
constexpr int kThreads = 256;
constexpr float kEps = 1e-6f;

struct ClipTensor {
  const char* in;
  char* out;
  int64_t n;
  int32_t dtype;
  int32_t chunk0;  // chunks of the tensors before it
};
struct ClipTable {
  int ntensors, nchunks;
  int part0, nparts;  // this launch's first partial, and the partials of all launches
  double max_norm;
  double* parts;
  float* norm;
  ClipTensor t[kMaxTensors];
};

__device__ __forceinline__ const ClipTensor& tensor_of(const ClipTable& tab, int chunk) {
  int lo = 0, hi = tab.ntensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].chunk0 <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return tab.t[lo];
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; i++) r += s[i];
  __syncthreads();
  return r;
}

__global__ void __launch_bounds__(kThreads) k_clip_norm(const __grid_constant__ ClipTable tab) {
  double sum = 0;
  for (int c = blockIdx.x; c < tab.nchunks; c += gridDim.x) {
    const ClipTensor& t = tensor_of(tab, c);
    const int64_t lo = (int64_t)(c - t.chunk0) * kChunk, hi = min(t.n, lo + kChunk);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
      const double g = (double)ld_as<float>(t.in, t.dtype, i);
      sum = fma(g, g, sum);
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) tab.parts[tab.part0 + blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) k_clip_scale(const __grid_constant__ ClipTable tab) {
  double sum = 0;
  for (int i = threadIdx.x; i < tab.nparts; i += kThreads) sum += tab.parts[i];
  const double norm = sqrt(block_sum(sum));
  const double ratio = tab.max_norm / (norm + (double)kEps);
  const float f = ratio < 1.0 || isnan(ratio) ? (float)ratio : 1.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) *tab.norm = (float)norm;
  for (int c = blockIdx.x; c < tab.nchunks; c += gridDim.x) {
    const ClipTensor& t = tensor_of(tab, c);
    const int64_t lo = (int64_t)(c - t.chunk0) * kChunk, hi = min(t.n, lo + kChunk);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) st_as<float>(t.out, t.dtype, i, f * ld_as<float>(t.in, t.dtype, i));
  }
}

}  // namespace

extern "C" {

int lc_clip_grad_norm(lc_tensor* outs, lc_tensor* norm_out, const lc_tensor* grads, int n, double max_norm) {
  LC_API_BEGIN
  LC_CHECK(n >= 0 && norm_out && (n == 0 || (outs && grads)), "clip_grad_norm: outs, norm and grads are required");
  LC_CHECK(max_norm >= 0, "clip_grad_norm: max_norm must be >= 0");
  struct Held {
    std::vector<LcTensor*> ts;
    std::vector<void*> mem;
    ~Held() {
      for (auto* t : ts) release(t);
      for (void* p : mem) dfree(p);
    }
  } held;
  std::vector<LcTensor*> in(n);
  int64_t bytes = 0;
  std::vector<int64_t> offset(n);
  for (int i = 0; i < n; i++) {
    in[i] = check(grads[i], "clip_grad_norm");
    LC_CHECK(in[i]->dtype == LC_F32 || is_half(in[i]->dtype),
             "clip_grad_norm: gradient " + std::to_string(i) + " must be f32, f16 or bf16, got " + dtype_name(in[i]->dtype));
    offset[i] = bytes;
    bytes += (in[i]->numel() * dtype_size(in[i]->dtype) + 255) / 256 * 256;
  }
  for (int i = 0; i < n; i++) {
    LcTensor* c = contiguous(in[i]);
    if (c != in[i]) held.ts.push_back(c);
    in[i] = c;
  }
  LcTensor* norm = alloc(LC_F32, {});
  held.ts.push_back(norm);
  LcTensor* all = alloc(LC_U8, {bytes});
  held.ts.push_back(all);
  std::vector<LcTensor*> out(n);
  for (int i = 0; i < n; i++) {
    const std::vector<int64_t> sh = in[i]->dims();
    std::vector<int64_t> st(sh.size());
    int64_t s = 1;
    for (int d = (int)sh.size() - 1; d >= 0; d--) st[d] = s, s *= sh[d];
    out[i] = view_of(all, sh, st, offset[i] / dtype_size(in[i]->dtype));
    out[i]->dtype = in[i]->dtype;
    held.ts.push_back(out[i]);
  }
  std::vector<ClipTable> tabs(1);
  auto fresh = [&]() { tabs.back().ntensors = tabs.back().nchunks = 0; };
  fresh();
  for (int i = 0; i < n; i++) {
    const int64_t chunks = (in[i]->numel() + kChunk - 1) / kChunk;
    if (!chunks) continue;
    if (tabs.back().ntensors == kMaxTensors || tabs.back().nchunks + chunks > INT32_MAX) {
      LC_CHECK(chunks <= INT32_MAX, "clip_grad_norm: a gradient is too large");
      tabs.emplace_back();
      fresh();
    }
    ClipTable& tab = tabs.back();
    tab.t[tab.ntensors++] = {in[i]->data(), out[i]->data(), in[i]->numel(), in[i]->dtype, tab.nchunks};
    tab.nchunks += (int)chunks;
  }
  int parts = 0;
  std::vector<int> grid;
  for (auto& tab : tabs) {
    tab.part0 = parts;
    grid.push_back(std::max(1, std::min(tab.nchunks, num_sms() * 8)));
    parts += grid.back();
  }
  double* pd = (double*)dmalloc((size_t)parts * 8);
  held.mem.push_back(pd);
  for (auto& tab : tabs) {
    tab.nparts = parts;
    tab.max_norm = max_norm;
    tab.parts = pd;
    tab.norm = (float*)norm->data();
  }
  for (size_t i = 0; i < tabs.size(); i++) k_clip_norm<<<grid[i], kThreads, 0, stream()>>>(tabs[i]);
  for (size_t i = 0; i < tabs.size(); i++) k_clip_scale<<<grid[i], kThreads, 0, stream()>>>(tabs[i]);
  LC_LAUNCHED(2 * (int)tabs.size());
  for (int i = 0; i < n; i++) outs[i] = handle(out[i]);
  *norm_out = handle(norm);
  held.ts.erase(std::remove_if(held.ts.begin(), held.ts.end(),
                               [&](LcTensor* t) { return t == norm || std::find(out.begin(), out.end(), t) != out.end(); }),
                held.ts.end());
  LC_API_END
}

}  // extern "C"
