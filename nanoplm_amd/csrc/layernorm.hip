// C ABI of the layer norm (include/nplm_layernorm.h): argument checks, choice of kernels, launches.
#include <hip/hip_runtime.h>

#include <limits.h>

#include <type_traits>

#include "../../include/nplm_layernorm.h"
#include "layernorm_kernels.h"

namespace nplm {
namespace ln {
namespace {

constexpr long long kMaxRows = (long long)INT_MAX - (1 << 20);
constexpr int kNumCU = 256;
constexpr int kMaxSum = 4096;         // rows whose gradients a lane adds up in fp32

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
// Lanes of a row or head, two or more: with eight or more, heads of 16 channels (131072 rows of 1024) took the forward 224 us and the backward 430 in place of 87 and 161.
int lanes_of(int n, int per_lane) {
    int g = 2;
    while (g * per_lane < n) g *= 2;
    return g;
}
// Channels of a lane.
int per_lane(int n) { return n > 512 ? 16 : 8; }
struct Grid {
    int gx, gy;
};
// Blocks: what the chip holds at once, each going through many rows; the backward has more of them where a lane would add up too many rows in fp32.
Grid grid_of(long long T, int heads, int G, bool bwd) {
    const int R = G > 256 ? 1 : 256 / G, rows = heads < R ? R / heads : 1, gy = heads < R ? 1 : (heads + R - 1) / R;
    const long long steps = (T + rows - 1) / rows, least = bwd ? (steps + kMaxSum - 1) / kMaxSum : 1;
    long long gx = ((bwd ? 4 : 8) * kNumCU + gy - 1) / gy;
    gx = gx < least ? least : gx;
    return {(int)(steps < gx ? steps : gx), gy};
}

int check(int64_t T, int32_t C, int32_t heads, int32_t act, int32_t wdt) {
    if (T < 0 || T > kMaxRows || C < 1 || heads < 1 || C % heads) return -NPLM_DWCONV_ESHAPE;
    for (int32_t t : {act, wdt})
        if (t != NPLM_DWCONV_F32 && t != NPLM_DWCONV_BF16) return -NPLM_DWCONV_EDTYPE;
    return C / heads > NPLM_LAYERNORM_MAX_GROUP || heads > NPLM_LAYERNORM_MAX_HEADS ? -NPLM_DWCONV_EUNSUPPORTED : 0;
}
int check_stride(const void* t, int64_t stride, int32_t C) { return t && (stride < C || stride > ((int64_t)1 << 40)) ? -NPLM_DWCONV_ESHAPE : 0; }

// fn(BF16, VEC, G, PL)
template <typename Fn> int dispatch(bool bf16, bool wide, int n, Fn fn) {
    auto with_g = [&](auto B, auto V) -> int {
        std::integral_constant<int, 8> p8;
        std::integral_constant<int, 16> p16;
        if (per_lane(n) == 8) {
            switch (lanes_of(n, 8)) {
                case 2: return fn(B, V, std::integral_constant<int, 2>{}, p8);
                case 4: return fn(B, V, std::integral_constant<int, 4>{}, p8);
                case 8: return fn(B, V, std::integral_constant<int, 8>{}, p8);
                case 16: return fn(B, V, std::integral_constant<int, 16>{}, p8);
                case 32: return fn(B, V, std::integral_constant<int, 32>{}, p8);
                default: return fn(B, V, std::integral_constant<int, 64>{}, p8);
            }
        }
        switch (lanes_of(n, 16)) {
            case 64: return fn(B, V, std::integral_constant<int, 64>{}, p16);
            case 128: return fn(B, V, std::integral_constant<int, 128>{}, p16);
            case 256: return fn(B, V, std::integral_constant<int, 256>{}, p16);
            case 512: return fn(B, V, std::integral_constant<int, 512>{}, p16);
            default: return fn(B, V, std::integral_constant<int, 1024>{}, p16);
        }
    };
    if (bf16) return wide ? with_g(std::true_type{}, std::integral_constant<int, 8>{}) : with_g(std::true_type{}, std::integral_constant<int, 1>{});
    return wide ? with_g(std::false_type{}, std::integral_constant<int, 4>{}) : with_g(std::false_type{}, std::integral_constant<int, 1>{});
}

}  // namespace
}  // namespace ln
}  // namespace nplm

using namespace nplm;
using namespace nplm::ln;

extern "C" {

int nplm_layernorm_fwd(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, const void* weight, const void* bias, float eps, void* y,
                       int64_t T, int32_t C, int32_t heads, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream) {
    if (int e = check(T, C, heads, act_dtype, w_dtype)) return e;
    if (flags & ~(NPLM_LAYERNORM_RMS | NPLM_LAYERNORM_SHARED)) return -NPLM_DWCONV_EFLAGS;
    if (T == 0) return 0;
    if (!x || !y || (bias && !weight)) return -NPLM_DWCONV_ENULL;
    for (int e : {check_stride(x, x_stride, C), check_stride(gate, gate_stride, C)})
        if (e) return e;
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16;
    const size_t e = bf16 ? 2 : 4, we = w_dtype == NPLM_DWCONV_BF16 ? 2 : 4;
    if (!aligned(x, e) || !aligned(gate, e) || !aligned(y, e) || !aligned(weight, we) || !aligned(bias, we)) return -NPLM_DWCONV_EALIGN;
    const int n = C / heads;
    const Args a{(const char*)x, (const char*)gate, nullptr, (long long)(x_stride * e), (long long)(gate_stride * e), 0, weight, bias, (char*)y, nullptr, nullptr,
                 eps, (int)T, C, heads, n, w_dtype == NPLM_DWCONV_BF16, (int)(flags & NPLM_LAYERNORM_RMS), (flags & NPLM_LAYERNORM_SHARED) != 0, 0};
    const bool wide = n % (bf16 ? 8 : 4) == 0 && ((uintptr_t)x | (uintptr_t)gate | (uintptr_t)y | (uintptr_t)a.xs | (uintptr_t)(gate ? a.gs : 0) |
                                                  (uintptr_t)weight | (uintptr_t)bias) % 16 == 0;
    return dispatch(bf16, wide, n, [&](auto B, auto V, auto G, auto P) {
        const Grid g = grid_of(T, heads, G.value, false);
        hipLaunchKernelGGL((fwd_kernel<B.value, V.value, G.value, P.value>), dim3(g.gx, g.gy), dim3(G.value > 256 ? G.value : 256), 0, (hipStream_t)stream, a);
        return (int)hipGetLastError();
    });
}

size_t nplm_layernorm_bwd_workspace_bytes(int64_t T, int32_t C, int32_t heads) {
    if (T < 1 || T > kMaxRows || C < 1 || heads < 1 || C % heads || C / heads > NPLM_LAYERNORM_MAX_GROUP || heads > NPLM_LAYERNORM_MAX_HEADS) return 0;
    const int n = C / heads;
    const Grid g = grid_of(T, heads, lanes_of(n, per_lane(n)), true);
    // (one weight for all heads: a row of n for each of gy as well, which C covers)
    const size_t shared = (size_t)g.gx * g.gy * n, own = (size_t)g.gx * C;
    return ((shared > own ? shared : own) * 2 * sizeof(float) + 255) / 256 * 256;
}

int nplm_layernorm_bwd(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, const void* dy, int64_t dy_stride, const void* weight,
                       const void* bias, float eps, void* dx, void* dgate, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                       int64_t T, int32_t C, int32_t heads, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream) {
    if (int e = check(T, C, heads, act_dtype, w_dtype)) return e;
    if (flags & ~(NPLM_LAYERNORM_RMS | NPLM_LAYERNORM_SHARED | NPLM_LAYERNORM_GRADS_BF16)) return -NPLM_DWCONV_EFLAGS;
    if ((bias || dweight || dbias) && !weight) return -NPLM_DWCONV_ENULL;
    if (T > 0 && (!x || !dy || !dx || (gate && !dgate))) return -NPLM_DWCONV_ENULL;
    for (int e : {check_stride(x, x_stride, C), check_stride(gate, gate_stride, C), check_stride(dy, dy_stride, C)})
        if (e && T > 0) return e;
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16, g_bf16 = flags & NPLM_LAYERNORM_GRADS_BF16, shared = flags & NPLM_LAYERNORM_SHARED;
    const size_t e = bf16 ? 2 : 4, we = w_dtype == NPLM_DWCONV_BF16 ? 2 : 4, ge = g_bf16 ? 2 : 4;
    for (const void* t : {x, gate, dy, (const void*)dx, (const void*)dgate})
        if (!aligned(t, e)) return -NPLM_DWCONV_EALIGN;
    if (!aligned(weight, we) || !aligned(bias, we) || !aligned(dweight, ge) || !aligned(dbias, ge)) return -NPLM_DWCONV_EALIGN;
    const int want = (dweight ? 1 : 0) | (dbias ? 2 : 0), n = C / heads, columns = shared ? n : C;
    if (T > 0 && want && (!workspace || !aligned(workspace, 256) || workspace_bytes < nplm_layernorm_bwd_workspace_bytes(T, C, heads))) return -NPLM_DWCONV_EWORKSPACE;
    int blocks = 0;
    if (T > 0) {
        const Args a{(const char*)x, (const char*)gate, (const char*)dy, (long long)(x_stride * e), (long long)(gate_stride * e), (long long)(dy_stride * e), weight,
                     bias, (char*)dx, (char*)dgate, (float*)workspace, eps, (int)T, C, heads, n, w_dtype == NPLM_DWCONV_BF16, (int)(flags & NPLM_LAYERNORM_RMS),
                     shared, want};
        const bool wide = n % (bf16 ? 8 : 4) == 0 && ((uintptr_t)x | (uintptr_t)gate | (uintptr_t)dy | (uintptr_t)dx | (uintptr_t)dgate | (uintptr_t)a.xs |
                                                      (uintptr_t)(gate ? a.gs : 0) | (uintptr_t)a.ds | (uintptr_t)weight | (uintptr_t)bias) % 16 == 0;
        const int err = dispatch(bf16, wide, n, [&](auto B, auto V, auto G, auto P) {
            const Grid g = grid_of(T, heads, G.value, true);
            blocks = shared ? g.gx * g.gy : g.gx;
            hipLaunchKernelGGL((bwd_kernel<B.value, V.value, G.value, P.value>), dim3(g.gx, g.gy), dim3(G.value > 256 ? G.value : 256), 0, (hipStream_t)stream, a);
            return (int)hipGetLastError();
        });
        if (err) return err;
    }
    if (!want) return 0;
    hipLaunchKernelGGL(sum_kernel, dim3((columns + 15) / 16, 2), dim3(1024), 0, (hipStream_t)stream, (const float*)workspace, dweight, dbias, blocks, columns, (int)g_bf16);
    return (int)hipGetLastError();
}

}  // extern "C"
