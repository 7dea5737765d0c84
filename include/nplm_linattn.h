/*
 * nplm_linattn.h — C ABI of linear attention with a decay for each head over packed sequences in libnplm_dwconv.so: forward, backward and a
 * single-token step, for AMD MI355X (gfx950).
 *
 * The operator
 * ------------
 *   q, k, dq, dk   : [T, H, dk] (packed tokens x heads x key channels)
 *   v, o, do, dv   : [T, H, dv]
 *   log_decay      : one number a head, or one a token and head: log a_t
 *   cu             : int32 [S+1] as in nplm_dwconv.h; zero-length sequences are legal anywhere
 *   initial, state : fp32 [S, H, dk, dv], the state a sequence begins with (NULL: zeros) and the one it ends with
 *
 *   S_t = a_t S_{t-1} + k_t v_t^T,    o_t = scale * q_t S_t
 *
 * per head, from a sequence's first row to its last one, or from its last row to its first one with NPLM_LINATTN_REVERSE. Nothing crosses a sequence
 * boundary, a NaN or Inf neither; within a sequence one reaches what reads it of o and of state, in the backward up to 63 rows of its head more, and any of its
 * sequence and head of dlog_decay. log_decay is meant to be 0 or less, -inf included (the state is forgotten; below -138 counts as that); values above 0 are
 * computed as they are and overflow as they do.
 *
 * Products are formed in the activations' type and summed in fp32; states are fp32. As operands of bf16 products scores, weighted by their decays, and the rows that
 * are added to the state are rounded to bf16 and the state that rows read keeps 16 bits; what the gradient of a bf16 log_decay comes from keeps 16 bits, and 24 where an
 * fp32 result depends on it (states handed out, gradients of initial states and of an fp32 log_decay).
 *
 * Conventions are those of nplm_dwconv.h (device pointers owned by the caller, asynchronous on `stream`, error codes and nplm_dwconv_strerror, results that
 * are run-to-run bit-identical, cu read on the device and held within [0, T]). Rows outside [cu[0], cu[S]) are one extra sequence on that side that begins with
 * zeros. q, k, v, do and log_decay have strides in elements from row to row and from head to head (any from 0 up; channels are adjacent), other tensors are
 * contiguous. No output may overlap an input. dk, dv <= NPLM_LINATTN_MAX_DIM (else -NPLM_DWCONV_EUNSUPPORTED, nothing launched);
 * H * (T / 64 + S + 2) must lie below 2^23, else -NPLM_DWCONV_ESHAPE.
 */
#ifndef NPLM_LINATTN_H
#define NPLM_LINATTN_H

#include "nplm_dwconv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NPLM_LINATTN_REVERSE 1u     /* from a sequence's last row to its first one */
#define NPLM_LINATTN_HEAD_DECAY 2u  /* log_decay [H] (g_row is not looked at; dlog_decay is [H]) */

/* Most channels of a key and of a value. */
#define NPLM_LINATTN_MAX_DIM 128

/* Longest stride of any tensor in elements. */
#define NPLM_LINATTN_MAX_STRIDE ((int64_t)1 << 36)

/* Most rows of a step that names slots. */
#define NPLM_LINATTN_MAX_SLOTS (1 << 16)

/*
 * Forward. q, k, v, o: act_dtype; log_decay: g_dtype. bounds: nplm_linattn_bounds_bytes() bytes, 256-byte aligned, contents irrelevant on entry (NULL where that
 * is 0); the states at the boundaries that long sequences are divided at, for the backward (a caller without one drops them). NPLM_LINATTN_... flags. state may be NULL.
 */
size_t nplm_linattn_bounds_bytes(int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act_dtype);
int nplm_linattn_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                     const int32_t* cu, const void* log_decay, int64_t g_row, int64_t g_head, float scale, const float* initial, void* o, float* state,
                     void* bounds, size_t bounds_bytes, int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act_dtype, int32_t g_dtype,
                     uint32_t flags, void* stream);

/*
 * Backward from the forward's inputs and its bounds, do and, where there are any, initial, dstate (fp32 [S, H, dk, dv], the gradient of state) and state (the
 * forward's; needed for dlog_decay beside dstate): dq, dk, dv (contiguous, act_dtype), dlog_decay ([T, H], or [H] with NPLM_LINATTN_HEAD_DECAY, g_dtype, fully
 * overwritten, NULL: not wanted) and dinitial (fp32 [S, H, dk, dv] or NULL). workspace: nplm_linattn_bwd_workspace_bytes() bytes, 256-byte aligned.
 */
size_t nplm_linattn_bwd_workspace_bytes(int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act_dtype);
int nplm_linattn_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                     const void* dout, int64_t do_row, int64_t do_head, const int32_t* cu, const void* log_decay, int64_t g_row, int64_t g_head, float scale,
                     const float* initial, const float* state, const float* dstate, const void* bounds, size_t bounds_bytes, void* dq, void* dk_out, void* dv_out,
                     void* dlog_decay, float* dinitial, void* workspace, size_t workspace_bytes, int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv,
                     int32_t act_dtype, int32_t g_dtype, uint32_t flags, void* stream);

/*
 * Step: row b of q, k [B, H, dk] and v [B, H, dv] is one token of the sequence whose state is row slots[b] (or b, slots NULL) of state [N, H, dk, dv]; its new
 * state goes to the same row of out_state (state itself, or another table apart from it, of which only the named rows are written), and scale * q S to row b of
 * o (contiguous). log_decay: [H] with NPLM_LINATTN_HEAD_DECAY, else [B, H]. Rows that name the same slot are tokens of one sequence, in order. A slot outside
 * [0, N) marks a padding row: it reads and writes no state and its o is 0. With slots B is at most NPLM_LINATTN_MAX_SLOTS: every row looks through all of them.
 */
int nplm_linattn_step(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                      const void* log_decay, int64_t g_row, int64_t g_head, float scale, const float* state, float* out_state, const int32_t* slots, void* o,
                      int64_t B, int32_t H, int64_t N, int32_t dk, int32_t dv, int32_t act_dtype, int32_t g_dtype, uint32_t flags, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* NPLM_LINATTN_H */
