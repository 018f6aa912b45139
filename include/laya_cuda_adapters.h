/*
 * liblaya_cuda — low-rank adapters of many requests beside a shared
 * projection, their gradients, and gradient clipping.
 *
 * One encoder serves many tenants: their requests share the projection W and
 * differ in a small adapter each. With s_a the scale (alpha / rank), A_a
 * [r, K] the down-projection and B_a [r, N] the up-projection of adapter a
 * (B_a is the transpose of the usual [N, r] matrix: both banks keep their
 * long axis contiguous, so every rank is served alike), row t of a batch gets
 *
 *   u[t] = s_a · A_a · x[t]                       a = the adapter of row t
 *   y[t] = W · x[t] (+ bias) + B_aᵀ · u[t]        rows without an adapter: W · x[t] (+ bias)
 *
 * The reference has no counterpart: its backends compute `linear`
 * (packages/tensor-backend/src/index.ts:211-215) alone. Conventions are those
 * of laya_cuda.h: int returns, lc_last_error(), handles, the library stream.
 */
#ifndef LAYA_CUDA_ADAPTERS_H
#define LAYA_CUDA_ADAPTERS_H
#include "laya_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The rows of one batch and the adapter of each request: request i owns rows
 * cu_rows[i] .. cu_rows[i + 1] (host, nseg + 1 entries from 0, not
 * decreasing; a request may be empty) and uses adapter adapters[i] (host,
 * -1 = none, else below n_adapters). Both arrays are copied before the call
 * returns. A plan serves every layer's projections of its batch; it is built
 * on the library stream, may be used on another (the use waits for the
 * build), and has to outlive the graphs recorded with it. At most 2^31 - 1024
 * rows.
 */
int lc_adapter_plan_create(uint64_t* plan, const int32_t* cu_rows, const int32_t* adapters, int nseg, int n_adapters);
int lc_adapter_plan_free(uint64_t plan);

/*
 * y = x·wᵀ (+ bias) + the adapters' share. x [..., K] with as many rows as
 * the plan; w [N, K], or 0 for the adapters' share alone (a shared projection
 * that is computed elsewhere, such as a packed one); bias [N] or 0;
 * a [n, r, K], b [n, r, N] and scales f32 [n] (0 = every scale 1) with
 * n = the plan's n_adapters. x, w, a and b share a dtype: f32, f16 or bf16.
 * Sums are held in f32 and rounded once, u as three bf16 parts that make up
 * the f32 value (all of its bits and range). No row's result depends on
 * another row or on another request's adapter, finite or not; a result that
 * depends on an inf or a NaN is one of the two (NaN also where f32 arithmetic
 * would keep an inf, since the parts of u meet it one by one).
 */
int lc_adapter_linear(lc_tensor* out, lc_tensor x, lc_tensor w, lc_tensor bias, lc_tensor a, lc_tensor b, lc_tensor scales, uint64_t plan);

/*
 * Gradients of adapter_linear for dy [..., N] (w, bias and scales are
 * frozen), each left out when its out-pointer is NULL:
 *   g[t] = s_a · B_a · dy[t]
 *   dx[t] = wᵀ · dy[t] + A_aᵀ · g[t]     [..., K]  (w = 0: the adapters' share)
 *   da_a = Σ_t g[t] ⊗ x[t]               [n, r, K]
 *   db_a = Σ_t u[t] ⊗ dy[t]              [n, r, N]
 * over the rows t of adapter a; an adapter without rows gets zeros. In the
 * inputs' dtype, summed in f32 in a fixed order (the same bits every run). u
 * and g are held as for adapter_linear; in the sums da and db of f16, whose
 * MMA takes f16 parts, exact to 2^-39 and up to 3.4e10 in magnitude.
 */
int lc_adapter_linear_grad(lc_tensor* dx, lc_tensor* da, lc_tensor* db, lc_tensor dy, lc_tensor x, lc_tensor w, lc_tensor a, lc_tensor b,
                           lc_tensor scales, uint64_t plan);

/*
 * Global-norm clipping of n gradient tensors (f32, f16 and bf16 in any mix,
 * any shapes): norm = sqrt(Σ g²) over all of them as an f32 scalar, and
 * outs[i] = grads[i] · min(1, max_norm / (norm + 1e-6)), in the order and
 * dtypes given. Squares are summed in f64 across threads, so neither a
 * gradient of 1e30 nor of 1e-30 is lost. A non-finite gradient shows in norm
 * (inf or NaN) and follows the same formula. max_norm >= 0, or inf (the norm
 * alone). The outputs share one allocation, released with the last of them.
 */
int lc_clip_grad_norm(lc_tensor* outs, lc_tensor* norm, const lc_tensor* grads, int n, double max_norm);

#ifdef __cplusplus
}
#endif
#endif /* LAYA_CUDA_ADAPTERS_H */
