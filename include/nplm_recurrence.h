/*
 * nplm_recurrence.h — C ABI of the gated linear recurrence over packed sequences in libnplm_dwconv.so: forward, backward and a
 * single-token step, for AMD MI355X (gfx950).
 *
 * The operator
 * ------------
 *   x, y, dy, dx   : [T, C] (packed tokens x channels)
 *   gates, dgates  : [T, 2C]: recurrence gate r in columns [0, C), input gate i in columns [C, 2C), both in front of their sigmoids
 *   cu             : int32 [S+1] as in nplm_dwconv.h; zero-length sequences are legal anywhere
 *   decay          : [C]
 *   initial, state : fp32 [S, C], the state a sequence begins with (NULL: zeros) and the one it ends with
 *
 *   z_t = scale * softplus(decay) * sigmoid(r_t),   a_t = exp(-z_t)
 *   h_t = a_t h_{t-1} + sqrt(1 - a_t^2) * sigmoid(i_t) * x_t,    y = h
 *
 * per channel, from a sequence's first row to its last one, or from its last row to its first one with NPLM_RECURRENCE_REVERSE (then
 * h_{t-1} reads h_{t+1}). Nothing crosses a sequence boundary, a NaN or Inf neither. Within a sequence an infinite state stays infinite, however little the
 * decays leave of it (where one of them is 0 in fp32, z above 103, it may be NaN). Everything is computed in fp32, 1 - a without cancellation; y, dx and dgates are
 * rounded once (nearest-even), states stay fp32.
 *
 * Conventions are those of nplm_dwconv.h (device pointers owned by the caller, asynchronous on `stream`, error codes and
 * nplm_dwconv_strerror, results that are run-to-run bit-identical, cu read on the device and used for masks and, checked against
 * [0, S), for rows of initial / state / dstate / dinitial). Rows outside [cu[0], cu[S]) are one extra sequence on that side that begins with zeros.
 * x, gates and dy have row strides in elements (any that their rows fit, up to NPLM_RECURRENCE_MAX_STRIDE), other tensors are contiguous. No output may overlap an input.
 * T * ceil(C / 128), in whole chunks, must lie below 2^29 in fp32 and 2^30 in bf16 (T itself up to 64 channels), else -NPLM_DWCONV_ESHAPE.
 */
#ifndef NPLM_RECURRENCE_H
#define NPLM_RECURRENCE_H

#include "nplm_dwconv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NPLM_RECURRENCE_REVERSE 1u    /* scan from a sequence's last row to its first one */
#define NPLM_RECURRENCE_GRADS_BF16 2u /* backward: ddecay points to a bf16 buffer */

/* Longest row stride, in elements, of any tensor; C is at most half of it. */
#define NPLM_RECURRENCE_MAX_STRIDE (1 << 24)

/* Most rows of a step that names slots. */
#define NPLM_RECURRENCE_MAX_SLOTS (1 << 18)

/* Rows of a chunk: the forward leaves the state in front of each chunk (in the scan's order) for the backward. */
#define NPLM_RECURRENCE_CHUNK 32

/*
 * Forward. carries: fp32 [ceil(T / NPLM_RECURRENCE_CHUNK), C] for the backward, or NULL. state may be NULL. x, gates, y: act_dtype;
 * decay: w_dtype. workspace: nplm_recurrence_fwd_workspace_bytes() bytes, 256-byte aligned, contents irrelevant on entry (NULL where that
 * is 0). T == 0 copies initial (or zeros) to state.
 */
size_t nplm_recurrence_fwd_workspace_bytes(int64_t T, int32_t C, int32_t S, int32_t act_dtype);
int nplm_recurrence_fwd(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const int32_t* cu, const void* decay,
                        float scale, const float* initial, void* y, float* state, float* carries, void* workspace, size_t workspace_bytes,
                        int64_t T, int32_t C, int32_t S, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream);

/*
 * Backward from x, gates, dy, the forward's carries and, where there are any, initial and dstate (fp32 [S, C], the gradient of state): dx,
 * dgates (contiguous [T, 2C]), ddecay (fp32 [C], or bf16 with NPLM_RECURRENCE_GRADS_BF16; summed over rows in fp32 and over chunks in fp64, in a
 * fixed order) and dinitial (fp32 [S, C] or NULL). T == 0 zero-fills ddecay and copies dstate (or zeros) to dinitial.
 */
size_t nplm_recurrence_bwd_workspace_bytes(int64_t T, int32_t C, int32_t S, int32_t act_dtype);
int nplm_recurrence_bwd(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const void* dy, int64_t dy_stride,
                        const int32_t* cu, const void* decay, float scale, const float* initial, const float* dstate, const float* carries,
                        void* dx, void* dgates, void* ddecay, float* dinitial, void* workspace, size_t workspace_bytes,
                        int64_t T, int32_t C, int32_t S, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream);

/*
 * Step: row b of x [B, C] and gates [B, 2C] is one token of the sequence whose state is row slots[b] (or b, slots NULL) of state [N, C];
 * its new state goes to the same row of out_state (which may be state itself, or another table, apart from it, of which only the named rows are
 * written) and, rounded to act_dtype, to row b of y. Rows that name the same slot are tokens of one sequence, in order. A slot outside [0, N) marks
 * a padding row: it reads and writes no state and its y is 0. B < 2^24, N <= 2^31 - 1; slots NULL needs B <= N.
 *
 * With slots every row looks through all B of them, and the first row of a slot that is named again goes on to the next one slot by slot: time grows with B squared, and
 * B is at most NPLM_RECURRENCE_MAX_SLOTS. C=2048, bf16, one MI355X, slots named once / each four times, at a distance of B / 4: B=512 9.9 / 69 us, 8192 0.30 / 6.8 ms,
 * 32768 3.3 / 105 ms (without slots 7.6 us, 76 us and as the bytes from there). Larger batches are better given in pieces.
 */
int nplm_recurrence_step(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const void* decay, float scale,
                         const float* state, float* out_state, const int32_t* slots, void* y,
                         int64_t B, int32_t C, int64_t N, int32_t act_dtype, int32_t w_dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NPLM_RECURRENCE_H */
