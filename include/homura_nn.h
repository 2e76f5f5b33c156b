/*
 * homura_nn.h -- the C ABI of libhomura_nn: operators of sequence models' recurrent blocks for gfx950, beside the
 * tensor path of homura_rocm.h. The reference has no counterpart of them, so they live in a library of their own and
 * the drop-in library keeps exporting exactly what the Rust crate declares.
 *
 *   hmn_recurrence   a gated linear recurrence over a sequence and its backward pass
 *   hmn_group_norm   group normalisation with an activation, channels last, and its backward pass
 *   hmn_dropout      dropout whose mask is computed from a counter, never stored; its backward pass is itself
 *
 * The conventions are homura_rocm.h's: contexts, tensor descriptions and status codes are the same, every entry point
 * returns an hmr_status, no exception leaves the library, the caller's current device is put back, and everything is
 * queued on the context's stream in the order of the calls. A failed call has queued nothing; its message is
 * hmn_last_error(), which belongs to the calling thread. No call allocates, waits, or keeps anything for the next one,
 * so all of them may be captured into a HIP graph (each replay computes from what the buffers hold then). Workspaces
 * are the caller's: device memory of at least 16-byte alignment whose contents do not matter, used only while the call's
 * kernels run, so that calls of one stream may share one and calls (or graphs) that may overlap need one each.
 *
 * Element types: F16, BF16, F32 and F64 tensors; F16, BF16 and F32 are computed in f32, F64 in f64, with one rounding to
 * the type at the end, except where said otherwise. Strides are any non-negative numbers of elements (outputs: no two
 * elements in one place); a channel stride of 1 is what the fast kernels want. Outputs share no memory with inputs
 * unless an entry point says so. Results repeat from run to run, bit for bit.
 */
#ifndef HOMURA_NN_H
#define HOMURA_NN_H

#include "homura_rocm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Text of the calling thread's most recent failure in this library ("" when it has had none). */
const char *hmn_last_error(void);

/* ---- gated linear recurrence ------------------------------------------------------------------------------------ */
/*
 * Over a batch of sequences [B, T, C], every channel by itself:
 *   GATE_FACTOR    h_t = gate_t * h_{t-1} + input_t
 *   GATE_SIGMOID   h_t = a_t * h_{t-1} + (1 - a_t) * input_t   with a_t = 1 / (1 + exp(-gate_t))
 * `out` gets every h_t; `last` [B, C], if not NULL, the state after the last step. `initial` [B, C] is the state before
 * the first (NULL: zero). `lengths` (1-D, B elements, I32 or I64; NULL: all of T) gives each sequence its own number
 * of steps, taken into 0..T: `last` is then the state after that many steps, and `out` behind them is zero whatever gate
 * and input hold there. The states are computed and carried in the computation type; `initial` and `last` may be F32
 * beside F16 or BF16 sequences (each for itself), so that a state handed from call to call is never rounded. `last` may
 * be `initial` itself. With T = 1 the call is one step of decoding, with T = 0 it copies the state.
 *
 * A scan folds stretches of steps into (product of factors, state from zero), so a product of factors beyond the
 * computation type's range is not finite where step-by-step evaluation might be, and one too small for it is zero. Factors
 * of magnitude at most one, as gates are, never meet the first, and the second loses nothing of a state in any ordinary
 * range. From a step with a factor that is itself not finite on, no state of the channel is finite; which ones are infinite
 * and which NaN depends on the grouping and may differ between `out` and `last`. The same holds backwards, from the end.
 */
#define HMN_GATE_FACTOR 0
#define HMN_GATE_SIGMOID 1

/* Workspace of both directions for sequences described as `gate` (its sizes and type). */
hmr_status hmn_recurrence_workspace(const hmr_tensor_desc *gate, int64_t *bytes);

hmr_status hmn_recurrence(hmr_context_t ctx, int32_t form, const hmr_tensor_desc *out,
                          const hmr_tensor_desc *last, const hmr_tensor_desc *gate,
                          const hmr_tensor_desc *input, const hmr_tensor_desc *initial,
                          const hmr_tensor_desc *lengths, void *workspace, int64_t workspace_bytes);

/*
 * The gradients of sum(grad * out) + sum(grad_last * last). `out` is what hmn_recurrence wrote and `input` may be NULL
 * for GATE_FACTOR (it isn't read). With g_t = grad_t + a_{t+1} g_{t+1} (a the factor; grad_last past the last step):
 *   GATE_FACTOR    d_input = g_t,             d_gate = g_t * h_{t-1}
 *   GATE_SIGMOID   d_input = (1 - a_t) g_t,   d_gate = g_t * (h_{t-1} - input_t) * a_t * (1 - a_t)
 * and d_initial = a_1 g_1. `grad_last`, `initial` and `d_initial` may be NULL (zero, zero, not wanted); the three states
 * may be F32 beside F16 or BF16 sequences, and so may `d_gate` (where one gate serves many channels or sequences, so that
 * their gradients are summed before they are rounded). Behind a sequence's length d_gate and d_input are zero and `grad` is not
 * read. d_initial may be grad_last itself.
 */
hmr_status hmn_recurrence_backward(hmr_context_t ctx, int32_t form, const hmr_tensor_desc *d_gate,
                                   const hmr_tensor_desc *d_input,
                                   const hmr_tensor_desc *d_initial, const hmr_tensor_desc *grad,
                                   const hmr_tensor_desc *grad_last, const hmr_tensor_desc *gate,
                                   const hmr_tensor_desc *input, const hmr_tensor_desc *out,
                                   const hmr_tensor_desc *initial, const hmr_tensor_desc *lengths,
                                   void *workspace, int64_t workspace_bytes);

/* ---- group normalisation with an activation ---------------------------------------------------------------------- */
/*
 * Channels last: `src` and `out` are [N, S, C] (S positions: pixels, or 1 for tokens), the C channels in `groups` equal
 * runs. For each n and group, over its S * C / groups elements, with the biased variance:
 *   hat = (src - mean) * rstd,  rstd = 1 / sqrt(variance + eps),  out = act(hat * weight + bias)
 * `weight` and `bias` [C] (NULL: one, zero) have src's type or F32; `mean` and `rstd` [N, groups] (NULL: not wanted) are
 * F32, or F64 for F64. Mean and variance are accumulated in f64. `activation` is HMN_ACTIVATION_NONE or one of
 * HMR_UNARY_RELU, _SILU, _GELU and _GELU_TANH. S = 0 leaves NaN in mean and rstd.
 */
#define HMN_ACTIVATION_NONE (-1)

hmr_status hmn_group_norm_workspace(const hmr_tensor_desc *src, int64_t groups, int32_t backward,
                                    int64_t *bytes);

hmr_status hmn_group_norm(hmr_context_t ctx, const hmr_tensor_desc *out, const hmr_tensor_desc *mean,
                          const hmr_tensor_desc *rstd, const hmr_tensor_desc *src,
                          const hmr_tensor_desc *weight, const hmr_tensor_desc *bias, int64_t groups,
                          double eps, int32_t activation, void *workspace, int64_t workspace_bytes);

/*
 * The gradients of sum(grad * out), from the mean and rstd that hmn_group_norm wrote. With z = hat * weight + bias,
 * d = grad * act'(z) and <.> the mean over a group's elements:
 *   d_bias = sum over n, s of d,  d_weight = sum over n, s of d * hat
 *   d_src = rstd * (weight * d - <weight * d> - hat * <weight * d * hat>)
 * d_weight and d_bias [C] may be NULL (not wanted) and have src's type or F32, each for itself.
 * The derivative of RELU at zero is zero.
 */
hmr_status hmn_group_norm_backward(hmr_context_t ctx, const hmr_tensor_desc *d_src,
                                   const hmr_tensor_desc *d_weight, const hmr_tensor_desc *d_bias,
                                   const hmr_tensor_desc *grad, const hmr_tensor_desc *src,
                                   const hmr_tensor_desc *mean, const hmr_tensor_desc *rstd,
                                   const hmr_tensor_desc *weight, const hmr_tensor_desc *bias,
                                   int64_t groups, int32_t activation, void *workspace,
                                   int64_t workspace_bytes);

/* ---- dropout ------------------------------------------------------------------------------------------------------ */
/*
 * out = residual + (kept ? src / (1 - p) : 0), without `residual` (NULL) the second term alone. Element i, in row-major
 * order, is kept when word i % 4 of the Philox4x32-10 block offset + i / 4 under `seed` (the blocks of
 * hmr_random_uniform) is at least round(p * 2^32); at p = 1 nothing is. A dropped element's src is not looked at (NaN
 * and infinities leave nothing). The mask is a function of (seed, offset, i) alone - not of layout, type or launch - so
 * the backward pass is the same call on the gradient: d_src = hmn_dropout(grad, NULL, p, seed, offset), d_residual =
 * grad. The caller reserves (elements + 3) / 4 blocks of its generator. `base`, if not NULL, is a 64-bit word of device
 * memory that is added to `offset` when the kernel runs: a captured graph that moves it on draws a new mask with every
 * replay. Operands have one type and the same sizes; input strides may be 0; `out` may be `src` or `residual` itself.
 */
hmr_status hmn_dropout(hmr_context_t ctx, const hmr_tensor_desc *out, const hmr_tensor_desc *src,
                       const hmr_tensor_desc *residual, double p, uint64_t seed, uint64_t offset,
                       const uint64_t *base);

#ifdef __cplusplus
}
#endif

#endif /* HOMURA_NN_H */
