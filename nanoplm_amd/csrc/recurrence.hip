// C ABI of the gated linear recurrence (include/nplm_recurrence.h): argument checks, choice of kernels, launches.
#include <hip/hip_runtime.h>

#include <limits.h>
#include <math.h>

#include "../../include/nplm_recurrence.h"
#include "recurrence_kernels.h"

namespace nplm {
namespace rec {
namespace {

constexpr long long kMaxRows = (long long)INT_MAX - (1 << 20);       // as nplm_dwconv.h: row arithmetic is int32 with slack

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

int check_sizes(int64_t T, int32_t C, int32_t S, int32_t act, int32_t wdt) {
    if (T < 0 || T > kMaxRows || C < 1 || S < 0 || C >= 1 << 28) return -NPLM_DWCONV_ESHAPE;
    if ((act != NPLM_DWCONV_F32 && act != NPLM_DWCONV_BF16) || (wdt != NPLM_DWCONV_F32 && wdt != NPLM_DWCONV_BF16)) return -NPLM_DWCONV_EDTYPE;
    return 0;
}
bool usable(float scale) { return scale > 0.f && scale < INFINITY; }
// a row of `width` elements fits its stride
int check_stride(int64_t stride, int64_t width) { return stride < width || stride > ((int64_t)1 << 40) ? -NPLM_DWCONV_ESHAPE : 0; }

// Two channels a lane where every row of every tensor lets pairs be loaded at once.
bool pairs(int E, int C, uintptr_t bits) { return C % 2 == 0 && bits % (2 * E) == 0; }

}  // namespace
}  // namespace rec
}  // namespace nplm

using namespace nplm;
using namespace nplm::rec;

#define NPLM_LAUNCH(KERNEL, GRID, BLOCK, ARGS)                                                        \
    do {                                                                                              \
        hipLaunchKernelGGL((KERNEL), GRID, dim3(BLOCK), 0, (hipStream_t)stream, ARGS);                \
        return (int)hipGetLastError();                                                                \
    } while (0)

extern "C" {

size_t nplm_recurrence_fwd_workspace_bytes(int64_t, int32_t, int32_t, int32_t) { return 0; }
size_t nplm_recurrence_bwd_workspace_bytes(int64_t, int32_t, int32_t, int32_t) { return 0; }

int nplm_recurrence_fwd(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const int32_t* cu, const void* decay,
                        float scale, const float* initial, void* y, float* state, float* carries, void* workspace, size_t workspace_bytes,
                        int64_t T, int32_t C, int32_t S, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream) {
    (void)workspace, (void)workspace_bytes;
    if (int e = check_sizes(T, C, S, act_dtype, w_dtype)) return e;
    if (!usable(scale)) return -NPLM_DWCONV_ESHAPE;
    if (flags & ~NPLM_RECURRENCE_REVERSE) return -NPLM_DWCONV_EFLAGS;
    if (T == 0 && (!state || S == 0)) return 0;
    if (!cu || !decay || (T > 0 && (!x || !gates || !y))) return -NPLM_DWCONV_ENULL;
    if (T > 0) {
        if (int e = check_stride(x_stride, C)) return e;
        if (int e = check_stride(gates_stride, 2 * (int64_t)C)) return e;
    }
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16;
    const size_t E = bf16 ? 2 : 4;
    if (!aligned(x, E) || !aligned(gates, E) || !aligned(y, E) || !aligned(decay, w_dtype == NPLM_DWCONV_BF16 ? 2 : 4) || !aligned(cu, 4) ||
        !aligned(initial, 4) || !aligned(state, 4) || !aligned(carries, 4)) return -NPLM_DWCONV_EALIGN;
    const FwdArgs a{(const char*)x, (const char*)gates, (long long)(x_stride * E), (long long)(gates_stride * E), cu, decay, initial, (char*)y,
                    state, carries, scale, (int)T, C, S, w_dtype == NPLM_DWCONV_BF16};
    const bool rev = flags & NPLM_RECURRENCE_REVERSE;
    const bool two = pairs(E, C, (uintptr_t)x | (uintptr_t)gates | (uintptr_t)y | (uintptr_t)a.xs | (uintptr_t)a.gs);
    const dim3 grid(ceil_div(C, two ? 128 : 64));
    if (bf16 && two && !rev) NPLM_LAUNCH((fwd_kernel<true, 2, 8, false>), grid, 512, a);
    if (bf16 && two) NPLM_LAUNCH((fwd_kernel<true, 2, 8, true>), grid, 512, a);
    if (bf16 && !rev) NPLM_LAUNCH((fwd_kernel<true, 1, 8, false>), grid, 512, a);
    if (bf16) NPLM_LAUNCH((fwd_kernel<true, 1, 8, true>), grid, 512, a);
    if (two && !rev) NPLM_LAUNCH((fwd_kernel<false, 2, 8, false>), grid, 512, a);
    if (two) NPLM_LAUNCH((fwd_kernel<false, 2, 8, true>), grid, 512, a);
    if (!rev) NPLM_LAUNCH((fwd_kernel<false, 1, 8, false>), grid, 512, a);
    NPLM_LAUNCH((fwd_kernel<false, 1, 8, true>), grid, 512, a);
}

int nplm_recurrence_bwd(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const void* dy, int64_t dy_stride,
                        const int32_t* cu, const void* decay, float scale, const float* initial, const float* dstate, const float* carries,
                        void* dx, void* dgates, void* ddecay, float* dinitial, void* workspace, size_t workspace_bytes,
                        int64_t T, int32_t C, int32_t S, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream) {
    (void)workspace, (void)workspace_bytes;
    if (int e = check_sizes(T, C, S, act_dtype, w_dtype)) return e;
    if (!usable(scale)) return -NPLM_DWCONV_ESHAPE;
    if (flags & ~(NPLM_RECURRENCE_REVERSE | NPLM_RECURRENCE_GRADS_BF16)) return -NPLM_DWCONV_EFLAGS;
    if (!cu || !decay || !ddecay || (T > 0 && (!x || !gates || !dy || !carries || !dx || !dgates))) return -NPLM_DWCONV_ENULL;
    if (T > 0) {
        if (int e = check_stride(x_stride, C)) return e;
        if (int e = check_stride(gates_stride, 2 * (int64_t)C)) return e;
        if (int e = check_stride(dy_stride, C)) return e;
    }
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16, g_bf16 = flags & NPLM_RECURRENCE_GRADS_BF16;
    const size_t E = bf16 ? 2 : 4;
    if (!aligned(x, E) || !aligned(gates, E) || !aligned(dy, E) || !aligned(dx, E) || !aligned(dgates, E) || !aligned(cu, 4) ||
        !aligned(decay, w_dtype == NPLM_DWCONV_BF16 ? 2 : 4) || !aligned(initial, 4) || !aligned(dstate, 4) || !aligned(carries, 4) ||
        !aligned(ddecay, g_bf16 ? 2 : 4) || !aligned(dinitial, 4)) return -NPLM_DWCONV_EALIGN;
    const BwdArgs a{(const char*)x, (const char*)gates, (const char*)dy, (long long)(x_stride * E), (long long)(gates_stride * E),
                    (long long)(dy_stride * E), cu, decay, initial, dstate, carries, (char*)dx, (char*)dgates, ddecay, dinitial, scale,
                    (int)T, C, S, w_dtype == NPLM_DWCONV_BF16, g_bf16};
    const bool rev = flags & NPLM_RECURRENCE_REVERSE;
    const bool two = pairs(E, C, (uintptr_t)x | (uintptr_t)gates | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)dgates | (uintptr_t)a.xs |
                                 (uintptr_t)a.gs | (uintptr_t)a.ds);
    const dim3 grid(ceil_div(C, two ? 128 : 64));
    if (bf16 && two && !rev) NPLM_LAUNCH((bwd_kernel<true, 2, 8, false>), grid, 512, a);
    if (bf16 && two) NPLM_LAUNCH((bwd_kernel<true, 2, 8, true>), grid, 512, a);
    if (bf16 && !rev) NPLM_LAUNCH((bwd_kernel<true, 1, 8, false>), grid, 512, a);
    if (bf16) NPLM_LAUNCH((bwd_kernel<true, 1, 8, true>), grid, 512, a);
    if (two && !rev) NPLM_LAUNCH((bwd_kernel<false, 2, 8, false>), grid, 512, a);
    if (two) NPLM_LAUNCH((bwd_kernel<false, 2, 8, true>), grid, 512, a);
    if (!rev) NPLM_LAUNCH((bwd_kernel<false, 1, 8, false>), grid, 512, a);
    NPLM_LAUNCH((bwd_kernel<false, 1, 8, true>), grid, 512, a);
}

int nplm_recurrence_step(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const void* decay, float scale,
                         const float* state, float* out_state, const int32_t* slots, void* y,
                         int64_t B, int32_t C, int64_t N, int32_t act_dtype, int32_t w_dtype, void* stream) {
    if (int e = check_sizes(B, C, 0, act_dtype, w_dtype)) return e;
    if (!usable(scale)) return -NPLM_DWCONV_ESHAPE;
    if (N < 0 || N > INT_MAX || (!slots && B > N)) return -NPLM_DWCONV_ESHAPE;
    if (B == 0) return 0;
    if (!x || !gates || !decay || !y || (N > 0 && (!state || !out_state))) return -NPLM_DWCONV_ENULL;
    if (int e = check_stride(x_stride, C)) return e;
    if (int e = check_stride(gates_stride, 2 * (int64_t)C)) return e;
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16;
    const size_t E = bf16 ? 2 : 4;
    if (!aligned(x, E) || !aligned(gates, E) || !aligned(y, E) || !aligned(decay, w_dtype == NPLM_DWCONV_BF16 ? 2 : 4) || !aligned(state, 4) ||
        !aligned(out_state, 4) || !aligned(slots, 4)) return -NPLM_DWCONV_EALIGN;
    const StepArgs a{(const char*)x, (const char*)gates, (long long)(x_stride * E), (long long)(gates_stride * E), decay, state, out_state,
                     slots, (char*)y, scale, (long long)N, (int)B, C, w_dtype == NPLM_DWCONV_BF16};
    const int cols = ceil_div(C, 256);
    if (cols > 65535) return -NPLM_DWCONV_ESHAPE;
    const dim3 grid((unsigned)B, cols);
    if (bf16) NPLM_LAUNCH((step_kernel<true>), grid, 256, a);
    NPLM_LAUNCH((step_kernel<false>), grid, 256, a);
}

}  // extern "C"
