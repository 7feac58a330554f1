/*
 * homura_cuda_layers.h: the trainable operators of a recurrent sequence block that are not one elementwise kernel or
 * one reduction: a gated linear recurrence, group norm with an activation (channels last) and dropout from the
 * counter-based generator, each forward and backward.
 *
 * homura has none of them (its layers are compositions of the operators of homura_cuda.h), so nothing here replaces a
 * declaration of csrc/homura_rocm.h; the rules of homura_cuda.h hold: status and message, the context's stream, the
 * thread's device restored, nothing queued by a failing call, workspaces from the caller, results that repeat bit for
 * bit (every sum is folded in an order fixed by sizes, dtypes and alignment). Arguments are checked before the context is
 * looked at.
 *
 * The descriptions here are not merged: they have exactly the dimensions named below, in that order, sizes of 1
 * included. Strides are any non-negative numbers of elements (an input may broadcast by a stride of 0, the elements of
 * an output are distinct) unless an entry says more. T is F16, BF16, F32 or F64; the computation type is f32, for F64
 * f64; each result is rounded to its dtype once. Optional descriptions are NULL when absent. A workspace is in use until
 * the call's kernels have run: a later call on the same context may take it again, calls that may run at the same time
 * (on two contexts, in two graphs) need one each.
 */
#ifndef HOMURA_CUDA_LAYERS_H
#define HOMURA_CUDA_LAYERS_H

#include "homura_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- gated linear recurrence ---- */
#define HMC_RECURRENCE_SIGMOID 1    /* the gate holds logits: a = sigmoid(gate); otherwise a = gate. F16 and BF16 logits g give
                                     * a and 1 - a to (12 + 2 |g|) 2^-24 of their values, and a = 0 below -87.3 */
#define HMC_RECURRENCE_COMPLEMENT 2 /* the input is weighted by what the gate leaves: u = (1 - a) * x; otherwise u = x */
#define HMC_RECURRENCE_REVERSE 4    /* time runs from the last row to the first */

/* h_t = a_t * h_{t-1} + u_t for every batch and channel. out, gate and x are [batch, time, channels] of one dtype T;
 * initial (h before the first step, zero when NULL) and last (receives h after the last step, unrounded; may be NULL
 * and may be the view `initial`) are [batch, channels] of F32 (F64 when T is F64). out may be the view x or the view
 * gate. The state is held in the computation type. A step with a = 0 forgets what came before it, whatever it was
 * unless that is infinite or NaN. With no time steps `last` receives `initial`. One step (time = 1) is the form for
 * generating a token. The time axis is folded in pieces of up to 128 steps: gates may exceed 1 in magnitude as long as
 * products of that many neighbours stay in the computation type's range. Where one overflows, a state of zero before the piece
 * still gives the right results, any other an infinity or NaN; where one underflows, less than the type's smallest number
 * times the state is lost. What an infinite state becomes where a product underflows or a gate is infinite is NaN or an
 * infinity. */
hmc_status hmc_linear_recurrence(hmc_context_t ctx, const hmc_tensor_desc *out, const hmc_tensor_desc *gate,
                                 const hmc_tensor_desc *x, const hmc_tensor_desc *initial, const hmc_tensor_desc *last,
                                 int32_t flags);

/* The gradients, with g_t = dout_t + a_{t+1} * g_{t+1} (g after the last step is dlast, zero when NULL):
 * dx_t = g_t (times 1 - a_t with COMPLEMENT), dgate_t = g_t * h_{t-1} (minus g_t * x_t with COMPLEMENT; times
 * a_t * (1 - a_t) with SIGMOID), dinitial = a_0 * g_0. `out` is what hmc_linear_recurrence wrote: h_{t-1} is read from
 * it (and from initial at the first step), so the gradients are those at the rounded states. x is read with COMPLEMENT
 * only and may be NULL otherwise; dinitial may be NULL. No output overlaps an input, except that dinitial may be the
 * view dlast. The flags are the forward call's. */
hmc_status hmc_linear_recurrence_backward(hmc_context_t ctx, const hmc_tensor_desc *dgate, const hmc_tensor_desc *dx,
                                          const hmc_tensor_desc *dinitial, const hmc_tensor_desc *gate,
                                          const hmc_tensor_desc *x, const hmc_tensor_desc *out,
                                          const hmc_tensor_desc *initial, const hmc_tensor_desc *dout,
                                          const hmc_tensor_desc *dlast, int32_t flags);

/* ---- group norm with an activation, channels last ---- */
#define HMC_ACTIVATION_NONE -1 /* otherwise HMC_UNARY_RELU, SILU, GELU or GELU_TANH */

/* out = act((src - mean) * rstd * weight + bias) where mean and rstd = 1 / sqrt(var + eps) are those of a group: the
 * channels / groups neighbouring channels of one sample at all its positions (var with divisor positions * channels /
 * groups). src and out are [samples, positions, channels] of T with a channel stride of 1 (or one channel); out may be
 * the view src. weight and bias (both or neither) are [channels] of T or of F32, alike. mean and rstd (both or neither)
 * receive the groups' moments, [samples, groups] of F32 (F64 when T is F64), for the backward pass. The moments are
 * taken in two passes over values held on chip: first the mean, then the deviations from it. Where a group is cut into
 * pieces, those are merged in f64, pairwise or (F16, BF16 and F32 in shared memory) through sums of n mean and n mean^2. A
 * piece's mean is rounded to the computation type before that, which does to the moments no more than rounding every element
 * once more would (2^-23 |mean| / deviation of the variance). A constant group becomes its bias as long as the sums of its elements are numbers of the computation
 * type. A NaN or an infinity makes its own group NaN, no other. The workspace has hmc_group_norm_workspace bytes
 * (0: NULL is fine), 16-byte aligned. */
hmc_status hmc_group_norm_workspace(const hmc_tensor_desc *src, int32_t groups, int32_t backward, int64_t *bytes);
hmc_status hmc_group_norm(hmc_context_t ctx, const hmc_tensor_desc *out, const hmc_tensor_desc *src,
                          const hmc_tensor_desc *weight, const hmc_tensor_desc *bias, const hmc_tensor_desc *mean,
                          const hmc_tensor_desc *rstd, int32_t groups, double eps, int32_t activation, void *workspace,
                          int64_t workspace_bytes);

/* The gradients from dout, src and the forward call's mean, rstd, weight, bias and activation: with xhat = (src - mean)
 * * rstd, dz = dout * act'(xhat * weight + bias) and p = dz * weight, dsrc = rstd * (p - mean(p) - xhat * mean(p * xhat))
 * over each group, dweight = the sum of dz * xhat and dbias = the sum of dz over samples and positions ([channels], the
 * dtype of weight, or of T or F32 without one; either may be NULL). dsrc may be the view dout or src. The workspace has
 * hmc_group_norm_workspace(.., backward = 1) bytes. */
hmc_status hmc_group_norm_backward(hmc_context_t ctx, const hmc_tensor_desc *dsrc, const hmc_tensor_desc *dweight,
                                   const hmc_tensor_desc *dbias, const hmc_tensor_desc *src, const hmc_tensor_desc *dout,
                                   const hmc_tensor_desc *mean, const hmc_tensor_desc *rstd,
                                   const hmc_tensor_desc *weight, const hmc_tensor_desc *bias, int32_t groups,
                                   int32_t activation, void *workspace, int64_t workspace_bytes);

/* ---- dropout ---- */

/* out_i = (residual_i +) keep_i * src_i / (1 - p), where element i (in row-major order of the logical positions, so that
 * the mask does not depend on the layout) is kept when word i % 4 of the Philox block offset + i / 4 under `seed`
 * (hmc_random_uniform's blocks) is at least p * 2^32 rounded to an integer. The mask is never stored: the gradient is
 * the same call on dout with the same seed and offset and without a residual. A call uses ceil(elements / 4) blocks. A
 * dropped element contributes 0 whatever it holds, NaN and infinities included. 0 <= p <= 1; with p = 1 every element
 * is dropped. Any number of (merged) dimensions; out may be the view src or the view residual. */
hmc_status hmc_dropout(hmc_context_t ctx, const hmc_tensor_desc *out, const hmc_tensor_desc *src,
                       const hmc_tensor_desc *residual, double p, uint64_t seed, uint64_t offset);

#ifdef __cplusplus
}
#endif

#endif /* HOMURA_CUDA_LAYERS_H */
