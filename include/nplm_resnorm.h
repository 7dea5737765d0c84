/*
 * nplm_resnorm.h — C ABI of the residual norm in libnplm_dwconv.so: the end of a block fused with the norm in front of the next one,
 * forward and backward, for AMD MI355X (gfx950).
 *
 * The operator, for every row of C channels
 * -----------------------------------------
 *   v      = norm(u) * post_weight + post_bias       (u itself without post_weight)
 *   v      = v * silu(gate)                          (with gate)
 *   out    = residual + scale * v                    (scale: [C]; 1 without it)
 *   normed = norm(out) * pre_weight + pre_bias       (with pre_weight; what the next block reads)
 *
 *   norm(a) = (a - mean(a)) / sqrt(var(a) + eps)     LayerNorm (biased variance), or, with NPLM_RESNORM_RMS,
 *             a / sqrt(mean(a^2) + eps)
 *
 * u, gate, normed, dnormed, du, dgate: [T, C], act_dtype. residual, out, dout, dresidual: [T, C], stream_dtype (the residual stream; act_dtype, or
 * fp32 beside bf16 branches, as torch.autocast leaves it). Parameters: [C], w_dtype. Everything is computed in fp32 and rounded once (nearest-even):
 * normed is formed from out before out is rounded.
 *
 * Conventions are those of nplm_dwconv.h (device pointers owned by the caller, asynchronous on `stream`, error codes and nplm_dwconv_strerror,
 * results that are run-to-run bit-identical). Inputs have row strides in elements (any that their rows fit), outputs are contiguous and overlap no
 * input. C <= NPLM_RESNORM_MAX_C (else -NPLM_DWCONV_EUNSUPPORTED, nothing launched).
 *
 * Where it sits in the reference (peymanvahidi/nanoplm 0.1.6): `x = x + sub_module(norm(x))` of the pre-norm encoder layer,
 * src/nanoplm/pretraining/models/modern_bert/modeling.py:404-438, from one sub-module's output to the next one's input.
 */
#ifndef NPLM_RESNORM_H
#define NPLM_RESNORM_H

#include "nplm_dwconv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NPLM_RESNORM_RMS 1u        /* root mean square instead of LayerNorm, in both places */
#define NPLM_RESNORM_GRADS_BF16 2u /* backward: the parameters' gradients point to bf16 buffers */

#define NPLM_RESNORM_MAX_C 16384

/*
 * Forward. gate, post_weight, post_bias, scale, pre_weight, pre_bias may be NULL; post_bias needs post_weight, pre_bias and normed need
 * pre_weight. stats: fp32 [T, 4] for the backward, (mean, 1 / sqrt(var + eps)) of u and of out, or NULL.
 */
int nplm_resnorm_fwd(const void* u, int64_t u_stride, const void* gate, int64_t gate_stride, const void* residual, int64_t residual_stride,
                     const void* post_weight, const void* post_bias, const void* scale, const void* pre_weight, const void* pre_bias, float eps,
                     void* out, void* normed, float* stats, int64_t T, int32_t C, int32_t act_dtype, int32_t stream_dtype, int32_t w_dtype,
                     uint32_t flags, void* stream);

/*
 * Backward from the forward's inputs, its stats and the gradients of out (NULL: zeros) and normed (NULL: zeros): du, dgate (with gate), dresidual, and
 * the gradients of the parameters that there are, fp32 (bf16 with NPLM_RESNORM_GRADS_BF16), fully overwritten, in a fixed order of sums; each of
 * them may be NULL. workspace: nplm_resnorm_bwd_workspace_bytes() bytes, 256-byte aligned, contents irrelevant on entry.
 */
size_t nplm_resnorm_bwd_workspace_bytes(int64_t T, int32_t C);
int nplm_resnorm_bwd(const void* u, int64_t u_stride, const void* gate, int64_t gate_stride, const void* residual, int64_t residual_stride,
                     const void* dout, int64_t dout_stride, const void* dnormed, int64_t dnormed_stride, const float* stats,
                     const void* post_weight, const void* post_bias, const void* scale, const void* pre_weight,
                     void* du, void* dgate, void* dresidual, void* dpost_weight, void* dpost_bias, void* dscale, void* dpre_weight, void* dpre_bias,
                     void* workspace, size_t workspace_bytes, int64_t T, int32_t C, int32_t act_dtype, int32_t stream_dtype, int32_t w_dtype,
                     uint32_t flags, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NPLM_RESNORM_H */
