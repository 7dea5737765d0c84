// C ABI of the gated linear recurrence (include/nplm_recurrence.h): argument checks, choice of kernels, launches.
#include <hip/hip_runtime.h>

#include <limits.h>
#include <math.h>

#include <type_traits>

#include "../../include/nplm_recurrence.h"
#include "recurrence_kernels.h"

namespace nplm {
namespace rec {
namespace {

constexpr long long kMaxRows = (long long)INT_MAX - (1 << 20);       // as nplm_dwconv.h: row arithmetic is int32 with slack

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

int check_sizes(int64_t T, int32_t C, int32_t S, int32_t act, int32_t wdt) {
    if (T < 0 || T > kMaxRows || C < 1 || S < 0 || 2 * (int64_t)C > NPLM_RECURRENCE_MAX_STRIDE) return -NPLM_DWCONV_ESHAPE;
    if ((act != NPLM_DWCONV_F32 && act != NPLM_DWCONV_BF16) || (wdt != NPLM_DWCONV_F32 && wdt != NPLM_DWCONV_BF16)) return -NPLM_DWCONV_EDTYPE;
    return 0;
}
bool usable(float scale) { return scale > 0.f && scale < INFINITY; }
// a row of `width` elements fits its stride, and a wave's rows 32-bit offsets
int check_stride(int64_t stride, int64_t width) { return stride < width || stride > NPLM_RECURRENCE_MAX_STRIDE ? -NPLM_DWCONV_ESHAPE : 0; }

// Channels of a lane: two, of whatever alignment (the hardware splits a word that lies in two lines; T=20011, C=1001, bf16: one channel a lane 65 and 134 us, two
// 58 and 112), one where that fills a wave (T=200000, C=16, bf16: 48 and 94 us, two 63 and 117). Below 64
// channels lanes lie idle: those 200000 rows take 44 and 89 us whether they have 16, 32 or 64 channels, whose bytes alone take 4 and 7, 8 and 14, 17 and 29.
int channels(int C) { return C > 64 ? 2 : 1; }

// Whether a wave's rows are whole cache lines, which it alone reads: its loads then go past the caches (nt). T=131072, C=1024, bf16: forward 255 -> 245 us, backward
// 525 -> 500; where two slices read a line (T=20011, C=1001) 58 -> 61 and 111 -> 114. (Stores go past them always: 261 and 541 us without. Parts of
// lines too: C=1001, one sequence, bf16, T=20011 59 and 110 us either way, T=50021 123 and 240, without 126 and 251; fp32, T=20011 84 and 155, without 86 and 167.)
bool whole_lines(size_t E, int C, uintptr_t bits) { return ((size_t)C * E | bits) % 128 == 0; }

// A launch counts its threads in 32 bits.
bool fits(int64_t T, int32_t C, const Shape& s) { return (long long)ceil_div(T, s.chunk()) * ceil_div(C, 64 * channels(C)) * s.waves * 64 <= (long long)UINT_MAX; }

// Where the board's parts lie in the workspace, and behind them K and the backward's sums. Sized for slices of 128 channels, the wider ones.
struct Layout {
    size_t tickets, pairs, groups, states, board, K, partial, all;
};
Layout layout(int64_t T, int32_t C, int chunk, bool bwd) {
    const size_t chunks = (T + chunk - 1) / chunk, width = ((size_t)C + 127) / 128 * 128;
    auto whole = [](size_t n) { return (n + 255) / 256 * 256; };
    Layout l;
    l.tickets = 0;
    l.pairs = whole(width / 64 * 64);
    l.groups = l.pairs + chunks * width * 8;
    l.states = l.groups + chunks / kGroup * width * 8;
    l.board = l.states + chunks / kSuper * width * 8;
    l.K = l.board;
    l.partial = l.K + whole((size_t)C * 4);
    l.all = l.partial + (bwd ? whole(chunks * C * 4) : 0);
    return l;
}
Board board_at(void* workspace, const Layout& l, int64_t T, int32_t C, int chunk, int V) {
    char* at = (char*)workspace;
    const int slices = ceil_div(C, 64 * V);
    return {(uint32_t*)(at + l.tickets), (uint64_t*)(at + l.pairs), (uint64_t*)(at + l.groups), (uint64_t*)(at + l.states), (float*)(at + l.K),
            ceil_div(T, chunk), slices * 64 * V, slices};
}
int prepare(const Board& b, const Layout& l, const void* decay, float scale, int C, int w_bf16, hipStream_t s) {
    const long long n = (long long)(l.board / 16), blocks = (n + 1023) / 1024;
    hipLaunchKernelGGL(prepare_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, (uint4*)b.tickets, n, b.K, decay, scale, C, w_bf16);
    return (int)hipGetLastError();
}
template <bool BF16, int V, bool REV, bool SPLIT, bool ONCE> struct Fwd {
    static int go(const FwdArgs& a, const Board& b, hipStream_t s) {
        const unsigned grid = SPLIT ? (unsigned)b.chunks * b.slices : ceil_div(a.C, 64 * V);
        hipLaunchKernelGGL((fwd_kernel<BF16, V, REV, SPLIT, ONCE>), dim3(grid), dim3(fwd_shape(BF16).waves * 64), 0, s, a, b);
        return (int)hipGetLastError();
    }
};
template <bool BF16, int V, bool REV, bool SPLIT, bool ONCE> struct Bwd {
    static int go(const BwdArgs& a, const Board& b, hipStream_t s) {
        const unsigned grid = SPLIT ? (unsigned)b.chunks * b.slices : ceil_div(a.C, 64 * V);
        hipLaunchKernelGGL((bwd_kernel<BF16, V, REV, SPLIT, ONCE>), dim3(grid), dim3(bwd_shape(BF16).waves * 64), 0, s, a, b);
        return (int)hipGetLastError();
    }
};
template <template <bool, int, bool, bool, bool> class Launch, typename Args>
int dispatch(bool bf16, bool rev, bool split, bool once, const Args& a, const Board& b, hipStream_t s) {
    auto with = [&](auto B, auto V, auto R) -> int {
        if (!split) return Launch<B.value, V.value, R.value, false, false>::go(a, b, s);
        if (V.value == 2 && once) return Launch<B.value, V.value, R.value, true, V.value == 2>::go(a, b, s);
        return Launch<B.value, V.value, R.value, true, false>::go(a, b, s);
    };
    auto with_v = [&](auto B, auto V) -> int { return rev ? with(B, V, std::true_type{}) : with(B, V, std::false_type{}); };
    auto with_b = [&](auto B) -> int {
        return channels(a.C) == 2 ? with_v(B, std::integral_constant<int, 2>{}) : with_v(B, std::integral_constant<int, 1>{});
    };
    return bf16 ? with_b(std::true_type{}) : with_b(std::false_type{});
}

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

size_t nplm_recurrence_fwd_workspace_bytes(int64_t T, int32_t C, int32_t S, int32_t act_dtype) {
    const Shape s = fwd_shape(act_dtype == NPLM_DWCONV_BF16);
    return check_sizes(T, C, S, act_dtype, 0) || T <= s.chunk() || !fits(T, C, s) ? 0 : layout(T, C, s.chunk(), false).all;
}
size_t nplm_recurrence_bwd_workspace_bytes(int64_t T, int32_t C, int32_t S, int32_t act_dtype) {
    const Shape s = bwd_shape(act_dtype == NPLM_DWCONV_BF16);
    return check_sizes(T, C, S, act_dtype, 0) || T <= s.chunk() || !fits(T, C, s) ? 0 : layout(T, C, s.chunk(), true).all;
}

int nplm_recurrence_fwd(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const int32_t* cu, const void* decay,
                        float scale, const float* initial, void* y, float* state, float* carries, void* workspace, size_t workspace_bytes,
                        int64_t T, int32_t C, int32_t S, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream) {
    if (int e = check_sizes(T, C, S, act_dtype, w_dtype)) return e;
    if (!usable(scale)) return -NPLM_DWCONV_ESHAPE;
    if (flags & ~NPLM_RECURRENCE_REVERSE) return -NPLM_DWCONV_EFLAGS;
    if (T == 0 && (!state || S == 0)) return 0;
    if (!cu || !decay || (T > 0 && (!x || !gates || !y))) return -NPLM_DWCONV_ENULL;
    if (T > 0) {
        if (int e = check_stride(x_stride, C)) return e;
        if (int e = check_stride(gates_stride, 2 * (int64_t)C)) return e;
    }
    if (!fits(T, C, fwd_shape(act_dtype == NPLM_DWCONV_BF16))) return -NPLM_DWCONV_ESHAPE;
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16;
    const size_t E = bf16 ? 2 : 4;
    if (!aligned(x, E) || !aligned(gates, E) || !aligned(y, E) || !aligned(decay, w_dtype == NPLM_DWCONV_BF16 ? 2 : 4) || !aligned(cu, 4) ||
        !aligned(initial, 4) || !aligned(state, 4) || !aligned(carries, 4)) return -NPLM_DWCONV_EALIGN;
    const FwdArgs a{(const char*)x, (const char*)gates, (long long)(x_stride * E), (long long)(gates_stride * E), cu, decay, initial, (char*)y,
                    state, carries, scale, (int)T, C, S, w_dtype == NPLM_DWCONV_BF16};
    const bool rev = flags & NPLM_RECURRENCE_REVERSE;
    const int chunk = fwd_shape(bf16).chunk();
    if (T <= chunk) return dispatch<Fwd>(bf16, rev, false, false, a, Board{}, (hipStream_t)stream);
    const bool once = whole_lines(E, C, (uintptr_t)x | (uintptr_t)gates | (uintptr_t)a.xs | (uintptr_t)a.gs);
    const Layout l = layout(T, C, chunk, false);
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.all) return -NPLM_DWCONV_EWORKSPACE;
    const Board b = board_at(workspace, l, T, C, chunk, channels(C));
    if (int e = prepare(b, l, decay, scale, C, a.w_bf16, (hipStream_t)stream)) return e;
    return dispatch<Fwd>(bf16, rev, true, once, a, b, (hipStream_t)stream);
}

int nplm_recurrence_bwd(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const void* dy, int64_t dy_stride,
                        const int32_t* cu, const void* decay, float scale, const float* initial, const float* dstate, const float* carries,
                        void* dx, void* dgates, void* ddecay, float* dinitial, void* workspace, size_t workspace_bytes,
                        int64_t T, int32_t C, int32_t S, int32_t act_dtype, int32_t w_dtype, uint32_t flags, void* stream) {
    if (int e = check_sizes(T, C, S, act_dtype, w_dtype)) return e;
    if (!usable(scale)) return -NPLM_DWCONV_ESHAPE;
    if (flags & ~(NPLM_RECURRENCE_REVERSE | NPLM_RECURRENCE_GRADS_BF16)) return -NPLM_DWCONV_EFLAGS;
    if (!cu || !decay || !ddecay || (T > 0 && (!x || !gates || !dy || !carries || !dx || !dgates))) return -NPLM_DWCONV_ENULL;
    if (T > 0) {
        if (int e = check_stride(x_stride, C)) return e;
        if (int e = check_stride(gates_stride, 2 * (int64_t)C)) return e;
        if (int e = check_stride(dy_stride, C)) return e;
    }
    if (!fits(T, C, bwd_shape(act_dtype == NPLM_DWCONV_BF16))) return -NPLM_DWCONV_ESHAPE;
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16, g_bf16 = flags & NPLM_RECURRENCE_GRADS_BF16;
    const size_t E = bf16 ? 2 : 4;
    if (!aligned(x, E) || !aligned(gates, E) || !aligned(dy, E) || !aligned(dx, E) || !aligned(dgates, E) || !aligned(cu, 4) ||
        !aligned(decay, w_dtype == NPLM_DWCONV_BF16 ? 2 : 4) || !aligned(initial, 4) || !aligned(dstate, 4) || !aligned(carries, 4) ||
        !aligned(ddecay, g_bf16 ? 2 : 4) || !aligned(dinitial, 4)) return -NPLM_DWCONV_EALIGN;
    BwdArgs a{(const char*)x, (const char*)gates, (const char*)dy, (long long)(x_stride * E), (long long)(gates_stride * E),
                    (long long)(dy_stride * E), cu, decay, initial, dstate, carries, (char*)dx, (char*)dgates, ddecay, dinitial, nullptr, scale,
                    (int)T, C, S, w_dtype == NPLM_DWCONV_BF16, g_bf16};
    const bool rev = flags & NPLM_RECURRENCE_REVERSE;
    const int chunk = bwd_shape(bf16).chunk();
    if (T <= chunk) return dispatch<Bwd>(bf16, rev, false, false, a, Board{}, (hipStream_t)stream);
    const bool once = whole_lines(E, C, (uintptr_t)x | (uintptr_t)gates | (uintptr_t)dy | (uintptr_t)a.xs | (uintptr_t)a.gs | (uintptr_t)a.ds);
    const Layout l = layout(T, C, chunk, true);
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < l.all) return -NPLM_DWCONV_EWORKSPACE;
    const Board b = board_at(workspace, l, T, C, chunk, channels(C));
    a.partial = (float*)((char*)workspace + l.partial);
    if (int e = prepare(b, l, decay, scale, C, a.w_bf16, (hipStream_t)stream)) return e;
    if (int e = dispatch<Bwd>(bf16, rev, true, once, a, b, (hipStream_t)stream)) return e;
    hipLaunchKernelGGL(sum_kernel, dim3(ceil_div(C, 16)), dim3(1024), 0, (hipStream_t)stream, a.partial, decay, ddecay, b.chunks, C, a.w_bf16, a.g_bf16);
    return (int)hipGetLastError();
}

int nplm_recurrence_step(const void* x, int64_t x_stride, const void* gates, int64_t gates_stride, const void* decay, float scale,
                         const float* state, float* out_state, const int32_t* slots, void* y,
                         int64_t B, int32_t C, int64_t N, int32_t act_dtype, int32_t w_dtype, void* stream) {
    if (int e = check_sizes(B, C, 0, act_dtype, w_dtype)) return e;
    if (!usable(scale)) return -NPLM_DWCONV_ESHAPE;
    if (B > (slots ? NPLM_RECURRENCE_MAX_SLOTS : (int64_t)UINT_MAX / 256) || N < 0 || N > INT_MAX || (!slots && B > N)) return -NPLM_DWCONV_ESHAPE;
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
