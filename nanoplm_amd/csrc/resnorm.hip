// C ABI of the residual norm (include/nplm_resnorm.h): argument checks, choice of kernels, launches.
#include <hip/hip_runtime.h>

#include <limits.h>

#include "../../include/nplm_resnorm.h"
#include "resnorm_kernels.h"

namespace nplm {
namespace rn {
namespace {

constexpr long long kMaxRows = (long long)INT_MAX - (1 << 20);
constexpr int kNumCU = 256;
constexpr int kMaxSum = 4096;         // rows whose gradients a lane adds up in fp32

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
int lanes_of(int C, int per_lane) {
    int g = 8;
    while (g * per_lane < C) g *= 2;
    return g;
}
// Channels of a lane. Up to 4096 channels (the forward in vectors: 8192) by what leaves two waves a SIMD their registers, in the backward with the parameters' five
// sums (T=131072, C=1024, bf16: 16 a lane 529 us, 8 456) and in rows that are loaded a channel at a time (forward, T=5003, C=1001, fp32: 22.6 and 19.5 us); else by
// fewer waves a row (forward 263 and 281). Wider rows are what a block of 1024 lanes can hold, four waves a SIMD with 128 registers: the backward spills 95 to 179
// of them up to 8192 channels and 508 to 605 beyond, the forward 102 to 300 beyond. 268 MB of bf16 a tensor, forward and backward: C=4096 264 and 541 us, 8192 240 and
// 1012, 16384 349 and 2759; fp32 248 and 411, 245 and 727, 346 and 1774.
constexpr int per_lane(int C, bool fwd, bool wide) { return C > 8 * 1024 || (fwd && wide) ? 16 : 8; }
// Rows that a block has at a time. Blocks: what the chip holds at once, each of them going through many rows with its parameters (forward 3 a CU 263 us, 8 a CU
// 277, 32 292; backward, as it was then, 2 a CU 434, 4 462, 1 623), more of them where a lane would add up too many rows in fp32.
long long rows_a_step(int lanes) { return lanes > 256 ? 1 : 256 / lanes; }
long long fwd_blocks(long long T, int lanes) {
    const long long steps = (T + rows_a_step(lanes) - 1) / rows_a_step(lanes), fill = 3 * kNumCU;
    return steps < fill ? steps : fill;
}
long long bwd_blocks(long long T, int C) {
    const long long rows = rows_a_step(lanes_of(C, per_lane(C, false, true))), steps = (T + rows - 1) / rows, least = (steps + kMaxSum - 1) / kMaxSum;
    const long long fill = 2 * kNumCU;
    return steps < fill ? steps : least > fill ? least : fill;
}

int check(int64_t T, int32_t C, int32_t act, int32_t st, int32_t wdt) {
    if (T < 0 || T > kMaxRows || C < 1) return -NPLM_DWCONV_ESHAPE;
    for (int32_t t : {act, st, wdt})
        if (t != NPLM_DWCONV_F32 && t != NPLM_DWCONV_BF16) return -NPLM_DWCONV_EDTYPE;
    if (act == NPLM_DWCONV_F32 && st == NPLM_DWCONV_BF16) return -NPLM_DWCONV_EDTYPE;      // (a stream narrower than its branches)
    return C > NPLM_RESNORM_MAX_C ? -NPLM_DWCONV_EUNSUPPORTED : 0;
}
int check_stride(const void* t, int64_t stride, int32_t C) { return t && (stride < C || stride > ((int64_t)1 << 40)) ? -NPLM_DWCONV_ESHAPE : 0; }

// Channels of a vector where rows allow it: 16 bytes of a tensor; of bf16 branches on an fp32 stream MIXED, 4 in the forward, whose stores then fill whole cache
// lines (T=50021, C=768: 111 us, 8 channels 120), and 8 in the backward, which has twice as many loads to ask for (as it was then 189, 4 channels 209).
template <template <bool, bool, int, int, int> class Launch, bool FWD, int MIXED, typename Args>
int dispatch(bool abf, bool sbf, bool wide, const Args& a, unsigned blocks, hipStream_t s) {
    auto with_g = [&](auto A, auto S, auto V) -> int {
        constexpr int PL = per_lane(1, FWD, V.value > 1);
        if constexpr (PL == 8)
            if (per_lane(a.C, FWD, wide) == 16) return Launch<A.value, S.value, V.value, 1024, 16>::go(a, blocks, s);
        switch (lanes_of(a.C, PL)) {
            case 8: return Launch<A.value, S.value, V.value, 8, PL>::go(a, blocks, s);
            case 16: return Launch<A.value, S.value, V.value, 16, PL>::go(a, blocks, s);
            case 32: return Launch<A.value, S.value, V.value, 32, PL>::go(a, blocks, s);
            case 64: return Launch<A.value, S.value, V.value, 64, PL>::go(a, blocks, s);
            case 128: return Launch<A.value, S.value, V.value, 128, PL>::go(a, blocks, s);
            case 256: return Launch<A.value, S.value, V.value, 256, PL>::go(a, blocks, s);
            case 512: return Launch<A.value, S.value, V.value, 512, PL>::go(a, blocks, s);
            default: return Launch<A.value, S.value, V.value, 1024, PL>::go(a, blocks, s);
        }
    };
    auto with_v = [&](auto A, auto S) -> int {
        return wide ? with_g(A, S, std::integral_constant<int, !A.value ? 4 : S.value ? 8 : MIXED>{}) : with_g(A, S, std::integral_constant<int, 1>{});
    };
    if (abf && sbf) return with_v(std::true_type{}, std::true_type{});
    if (abf) return with_v(std::true_type{}, std::false_type{});
    return with_v(std::false_type{}, std::false_type{});
}
template <bool A, bool S, int V, int G, int PL> struct Fwd {
    static int go(const FwdArgs& a, unsigned blocks, hipStream_t s) {
        hipLaunchKernelGGL((fwd_kernel<A, S, V, G, PL>), dim3(blocks), dim3(G > 256 ? G : 256), 0, s, a);
        return (int)hipGetLastError();
    }
};
template <bool A, bool S, int V, int G, int PL> struct Bwd {
    static int go(const BwdArgs& a, unsigned blocks, hipStream_t s) {
        hipLaunchKernelGGL((bwd_kernel<A, S, V, G, PL>), dim3(blocks), dim3(G > 256 ? G : 256), 0, s, a);
        return (int)hipGetLastError();
    }
};

}  // namespace
}  // namespace rn
}  // namespace nplm

using namespace nplm;
using namespace nplm::rn;

extern "C" {

int nplm_resnorm_fwd(const void* u, int64_t u_stride, const void* gate, int64_t gate_stride, const void* residual, int64_t residual_stride,
                     const void* post_weight, const void* post_bias, const void* scale, const void* pre_weight, const void* pre_bias, float eps,
                     void* out, void* normed, float* stats, int64_t T, int32_t C, int32_t act_dtype, int32_t stream_dtype, int32_t w_dtype,
                     uint32_t flags, void* stream) {
    if (int e = check(T, C, act_dtype, stream_dtype, w_dtype)) return e;
    if (flags & ~NPLM_RESNORM_RMS) return -NPLM_DWCONV_EFLAGS;
    if (T == 0) return 0;
    if (!u || !residual || !out || (post_bias && !post_weight) || ((pre_bias || normed) && !pre_weight)) return -NPLM_DWCONV_ENULL;
    for (int e : {check_stride(u, u_stride, C), check_stride(gate, gate_stride, C), check_stride(residual, residual_stride, C)})
        if (e) return e;
    const bool abf = act_dtype == NPLM_DWCONV_BF16, sbf = stream_dtype == NPLM_DWCONV_BF16;
    const size_t ae = abf ? 2 : 4, se = sbf ? 2 : 4, we = w_dtype == NPLM_DWCONV_BF16 ? 2 : 4;
    for (const void* t : {u, gate, (const void*)normed})
        if (!aligned(t, ae)) return -NPLM_DWCONV_EALIGN;
    for (const void* t : {post_weight, post_bias, scale, pre_weight, pre_bias})
        if (!aligned(t, we)) return -NPLM_DWCONV_EALIGN;
    if (!aligned(residual, se) || !aligned(out, se) || !aligned(stats, 16)) return -NPLM_DWCONV_EALIGN;
    const FwdArgs a{(const char*)u, (const char*)gate, (const char*)residual, (long long)(u_stride * ae), (long long)(gate_stride * ae),
                    (long long)(residual_stride * se), {post_weight, post_bias, scale, pre_weight, pre_bias}, (char*)out, (char*)normed, stats, eps,
                    (int)T, C, w_dtype == NPLM_DWCONV_BF16, (int)(flags & NPLM_RESNORM_RMS)};
    const bool wide = C % (abf ? 8 : 4) == 0 && ((uintptr_t)u | (uintptr_t)gate | (uintptr_t)residual | (uintptr_t)out | (uintptr_t)normed | (uintptr_t)a.us |
                                     (uintptr_t)(gate ? a.gs : 0) | (uintptr_t)a.rs | (uintptr_t)post_weight | (uintptr_t)post_bias | (uintptr_t)scale |
                                     (uintptr_t)pre_weight | (uintptr_t)pre_bias) % 16 == 0;
    const unsigned blocks = (unsigned)fwd_blocks(T, lanes_of(C, per_lane(C, true, wide)));
    return dispatch<Fwd, true, 4>(abf, sbf, wide, a, blocks, (hipStream_t)stream);
}

size_t nplm_resnorm_bwd_workspace_bytes(int64_t T, int32_t C) {
    if (T < 1 || T > kMaxRows || C < 1 || C > NPLM_RESNORM_MAX_C) return 0;
    return ((size_t)bwd_blocks(T, C) * kParams * C * sizeof(float) + 255) / 256 * 256;
}

int nplm_resnorm_bwd(const void* u, int64_t u_stride, const void* gate, int64_t gate_stride, const void* residual, int64_t residual_stride,
                     const void* dout, int64_t dout_stride, const void* dnormed, int64_t dnormed_stride, const float* stats,
                     const void* post_weight, const void* post_bias, const void* scale, const void* pre_weight,
                     void* du, void* dgate, void* dresidual, void* dpost_weight, void* dpost_bias, void* dscale, void* dpre_weight, void* dpre_bias,
                     void* workspace, size_t workspace_bytes, int64_t T, int32_t C, int32_t act_dtype, int32_t stream_dtype, int32_t w_dtype,
                     uint32_t flags, void* stream) {
    if (int e = check(T, C, act_dtype, stream_dtype, w_dtype)) return e;
    if (flags & ~(NPLM_RESNORM_RMS | NPLM_RESNORM_GRADS_BF16)) return -NPLM_DWCONV_EFLAGS;
    if (((dpost_weight || dpost_bias || post_bias) && !post_weight) || ((dpre_weight || dpre_bias || dnormed) && !pre_weight) || (dscale && !scale))
        return -NPLM_DWCONV_ENULL;
    if (T > 0 && (!u || !residual || !du || !dresidual || (gate && !dgate) || !stats)) return -NPLM_DWCONV_ENULL;
    for (int e : {check_stride(u, u_stride, C), check_stride(gate, gate_stride, C), check_stride(residual, residual_stride, C),
                  check_stride(dout, dout_stride, C), check_stride(dnormed, dnormed_stride, C)})
        if (e && T > 0) return e;
    const bool abf = act_dtype == NPLM_DWCONV_BF16, sbf = stream_dtype == NPLM_DWCONV_BF16, g_bf16 = flags & NPLM_RESNORM_GRADS_BF16;
    const size_t ae = abf ? 2 : 4, se = sbf ? 2 : 4, we = w_dtype == NPLM_DWCONV_BF16 ? 2 : 4;
    for (const void* t : {u, gate, dnormed, (const void*)du, (const void*)dgate})
        if (!aligned(t, ae)) return -NPLM_DWCONV_EALIGN;
    for (const void* t : {residual, dout, (const void*)dresidual})
        if (!aligned(t, se)) return -NPLM_DWCONV_EALIGN;
    for (const void* t : {post_weight, post_bias, scale, pre_weight})
        if (!aligned(t, we)) return -NPLM_DWCONV_EALIGN;
    void* const grads[kParams] = {dpost_weight, dpost_bias, dscale, dpre_weight, dpre_bias};
    int want = 0;
    for (int i = 0; i < kParams; ++i) {
        if (!aligned(grads[i], g_bf16 ? 2 : 4)) return -NPLM_DWCONV_EALIGN;
        want |= (grads[i] ? 1 : 0) << i;
    }
    if (!aligned(stats, 16)) return -NPLM_DWCONV_EALIGN;
    if (T > 0 && want && (!workspace || !aligned(workspace, 256) || workspace_bytes < nplm_resnorm_bwd_workspace_bytes(T, C))) return -NPLM_DWCONV_EWORKSPACE;
    const long long blocks = T > 0 ? bwd_blocks(T, C) : 0;
    if (T > 0) {
        const BwdArgs a{(const char*)u, (const char*)gate, (const char*)residual, (const char*)dout, (const char*)dnormed, (long long)(u_stride * ae),
                        (long long)(gate_stride * ae), (long long)(residual_stride * se), (long long)(dout_stride * se), (long long)(dnormed_stride * ae),
                        stats, {post_weight, post_bias, scale, pre_weight, nullptr}, (char*)du, (char*)dgate, (char*)dresidual, (float*)workspace,
                        (int)T, C, w_dtype == NPLM_DWCONV_BF16, (int)(flags & NPLM_RESNORM_RMS), want};
        const bool wide = C % (abf ? 8 : 4) == 0 && ((uintptr_t)u | (uintptr_t)gate | (uintptr_t)residual | (uintptr_t)dout | (uintptr_t)dnormed | (uintptr_t)du |
                                         (uintptr_t)dgate | (uintptr_t)dresidual | (uintptr_t)a.us | (uintptr_t)(gate ? a.gs : 0) | (uintptr_t)a.rs |
                                         (uintptr_t)(dout ? a.os : 0) | (uintptr_t)(dnormed ? a.ns : 0) | (uintptr_t)post_weight | (uintptr_t)post_bias |
                                         (uintptr_t)scale | (uintptr_t)pre_weight) % 16 == 0;
        if (int e = dispatch<Bwd, false, 8>(abf, sbf, wide, a, (unsigned)blocks, (hipStream_t)stream)) return e;
    }
    if (!want) return 0;
    const SumArgs a{(const float*)workspace, {grads[0], grads[1], grads[2], grads[3], grads[4]}, (int)blocks, C, g_bf16};
    hipLaunchKernelGGL(sum_kernel, dim3((C + 15) / 16, kParams), dim3(1024), 0, (hipStream_t)stream, a);
    return (int)hipGetLastError();
}

}  // extern "C"
