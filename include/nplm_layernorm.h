/*
 * nplm_layernorm.h — C ABI of the layer norm over rows or over each head's channels in libnplm_dwconv.so, forward and backward, for AMD MI355X (gfx950).
 *
 * The operator, for every row of C channels and each of its `heads` groups of C / heads adjacent ones
 * -----------------------------------------------------------------------------------------------
 *   y = (norm(x) * weight + bias) * silu(gate)          (weight 1, bias 0, no gate where they are NULL)
 *
 *   norm(a) = (a - mean(a)) / sqrt(var(a) + eps)        LayerNorm (biased variance), or, with NPLM_LAYERNORM_RMS,
 *             a / sqrt(mean(a^2) + eps)                  over the group's channels
 *
 * x, gate, y, dy, dx, dgate: [T, C], act_dtype. weight, bias: w_dtype, [C], or [C / heads] for all heads with NPLM_LAYERNORM_SHARED. Everything is computed in
 * fp32 and rounded once (nearest-even); the gradients of weight and bias are summed in fp32 over up to 4096 rows a lane and in fp64 from there, in a fixed order.
 *
 * Conventions are those of nplm_dwconv.h (device pointers owned by the caller, asynchronous on `stream`, error codes and nplm_dwconv_strerror, results that
 * are run-to-run bit-identical). Inputs have row strides in elements (any that their rows fit), outputs are contiguous and overlap no input.
 * heads divides C, heads <= NPLM_LAYERNORM_MAX_HEADS and C / heads <= NPLM_LAYERNORM_MAX_GROUP (else -NPLM_DWCONV_EUNSUPPORTED, nothing launched).
 *
 * Where it sits in the reference (peymanvahidi/nanoplm 0.1.6): the norms that stand alone, in front of the first layer and behind the last one
 * (src/nanoplm/pretraining/models/modern_bert/modeling.py:404-438 has those inside a layer).
 */
#ifndef NPLM_LAYERNORM_H
#define NPLM_LAYERNORM_H

#include "nplm_dwconv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NPLM_LAYERNORM_RMS 1u        /* root mean square instead of LayerNorm */
#define NPLM_LAYERNORM_GRADS_BF16 2u /* backward: dweight and dbias point to bf16 buffers */
#define NPLM_LAYERNORM_SHARED 4u     /* weight and bias are [C / heads] */

#define NPLM_LAYERNORM_MAX_GROUP 16384
#define NPLM_LAYERNORM_MAX_HEADS 65535

/* Forward. gate, weight and bias may be NULL; bias needs weight. */
int nplm_layernorm_fwd(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, const void* weight, const void* bias, float eps, void* y,
                       int64_t T, int32_t C, int32_t heads, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream);

/*
 * Backward from the forward's inputs and dy: dx, dgate (with gate), dweight and dbias (fp32, bf16 with NPLM_LAYERNORM_GRADS_BF16, fully overwritten; each of
 * them may be NULL). workspace: nplm_layernorm_bwd_workspace_bytes() bytes, 256-byte aligned, contents irrelevant on entry; needed for dweight and dbias.
 */
size_t nplm_layernorm_bwd_workspace_bytes(int64_t T, int32_t C, int32_t heads);
int nplm_layernorm_bwd(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, const void* dy, int64_t dy_stride, const void* weight,
                       const void* bias, float eps, void* dx, void* dgate, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                       int64_t T, int32_t C, int32_t heads, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NPLM_LAYERNORM_H */
