// C ABI of linear attention with a decay for each head (include/nplm_linattn.h): argument checks, choice of kernels, launches.
#include <hip/hip_runtime.h>

#include <limits.h>

#include <type_traits>

#include "../../include/nplm_linattn.h"
#include "linattn_kernels.h"

namespace nplm {
namespace la {
namespace {

constexpr long long kMaxRows = (long long)INT_MAX - (1 << 20);
constexpr long long kMaxBlocks = 1 << 23;

bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
size_t elem(int32_t t) { return t == NPLM_DWCONV_BF16 ? 2 : 4; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Rows of a segment: as few (of whole chunks, 64 to 2048) as make at most 512 blocks, two a CU. That is what the backward of 64 x 64 and of 128 channels of keys has on the chip at once;
// the rule does not look at what other kernels have (backward: 64 x 128 one, so that 512 are two rounds, up to 32 channels four; forward: 64 x 64 four, 64 x 128
// two). Its number was found on one shape, 20011 rows of 8 heads of 64 and 128 in one sequence, forward and backward with the kernels of then: 256 rows, 632 blocks, 302 us; 320
// rows, 504 blocks, 256 us. Where the sequences alone are more blocks than that, they are cut where they have more than 2048 rows. A small batch of short sequences
// goes without boundaries: fewer rows at a time, but 3 launches in place of 7 (776 rows of 10 sequences, 2 heads of 32, forward and backward: 61 us either way). What counts
// as short is the mean with empty sequences: 2048 rows of 2 heads of 64 in one, with 15 empty ones behind it, take 86 and 257 us, with 14 (segments of 64 rows) 23 and 35.
int segment_rows(int64_t T, int32_t H, int32_t S) {
    constexpr int kMost = 2048, kBlocks = 512;
    if (T <= kMost && T <= 128ll * S) return kMost;
    const long long left = kBlocks - (long long)S * H;
    if (left <= 0) return kMost;
    const long long L = (T * H + 64 * left - 1) / (64 * left) * 64;
    return L < 64 ? 64 : L > kMost ? kMost : (int)L;
}
long long slots_of(int64_t T, int32_t S, int L) { return T / L + S + 2; }
size_t state_bytes(int64_t T, int32_t H, int L, int32_t dk, int32_t dv) { return up256((size_t)(T / L + 1) * H * dk * dv * sizeof(float)); }
size_t decay_bytes(int64_t T, int32_t H, int L) { return up256((size_t)(T / L + 1) * H * sizeof(float)); }

int check_sizes(int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act, int32_t gdt) {
    if (T < 0 || T > kMaxRows || H < 1 || S < 0 || dk < 1 || dv < 1) return -NPLM_DWCONV_ESHAPE;
    for (int32_t t : {act, gdt})
        if (t != NPLM_DWCONV_F32 && t != NPLM_DWCONV_BF16) return -NPLM_DWCONV_EDTYPE;
    if (dk > NPLM_LINATTN_MAX_DIM || dv > NPLM_LINATTN_MAX_DIM) return -NPLM_DWCONV_EUNSUPPORTED;
    return (T / 64 + S + 2) * (int64_t)H < kMaxBlocks ? 0 : -NPLM_DWCONV_ESHAPE;
}
int check_tensor(const void* p, int64_t row, int64_t head, int32_t dt) {
    if (!p) return -NPLM_DWCONV_ENULL;
    if (row < 0 || head < 0 || row > NPLM_LINATTN_MAX_STRIDE || head > NPLM_LINATTN_MAX_STRIDE) return -NPLM_DWCONV_ESHAPE;
    return aligned(p, elem(dt)) ? 0 : -NPLM_DWCONV_EALIGN;
}
Tensor3 tensor(const void* p, int64_t row, int64_t head, int32_t d, int32_t dt) {
    const size_t e = elem(dt);
    const bool vec = d * e % 16 == 0 && ((uintptr_t)p | (uintptr_t)(row * e) | (uintptr_t)(head * e)) % 16 == 0;
    return {(const char*)p, (long long)(row * e), (long long)(head * e), vec};
}
Shape shape(const int32_t* cu, const void* g, int64_t g_row, int64_t g_head, int64_t T, int32_t H, int32_t S, int L, int32_t gdt, uint32_t flags) {
    const size_t e = elem(gdt);
    return {cu, (const char*)g, flags & NPLM_LINATTN_HEAD_DECAY ? 0 : (long long)(g_row * e), (long long)(g_head * e), gdt == NPLM_DWCONV_BF16, (int)T, H, S, L,
            (int)(flags & NPLM_LINATTN_REVERSE)};
}

// fn(BF16, VEC, DK, DV) of the kernels' sizes
template <typename Fn> int with_sizes(bool bf16, bool vec, int dk, int dv, Fn fn) {
    std::integral_constant<int, 32> t;
    std::integral_constant<int, 64> s;
    std::integral_constant<int, 128> b;
    auto go = [&](auto B, auto V) { return dk <= 32 && dv <= 32 ? fn(B, V, t, t) : dk <= 64 ? (dv <= 64 ? fn(B, V, s, s) : fn(B, V, s, b)) : dv <= 64 ? fn(B, V, b, s) : fn(B, V, b, b); };
    auto of = [&](auto B) { return vec ? go(B, std::true_type{}) : go(B, std::false_type{}); };
    return bf16 ? of(std::true_type{}) : of(std::false_type{});
}
int launched() { return (int)hipGetLastError(); }

// A segment's rows of a tensor within one buffer whose offsets 30 bits hold (Rows), every 16 bytes of it one load.
bool as_buffer(const Tensor3& t, int d, size_t e, int L) { return t.vec && t.row >= (long long)(d * e) && t.row * (L + 64) < (1ll << 30); }
// The same of a contiguous [T, H, d] that is written in fours.
bool out_as_buffer(int H, int d, size_t e, int L) { return d % 4 == 0 && (long long)H * d * (long long)e * (L + 64) < (1ll << 30); }

// terms: of the state as an operand (Split; fp32 activations have one)
int walk(const WalkArgs& a, bool bf16, int terms, bool dg, hipStream_t stream) {
    const unsigned blocks = (unsigned)(slots_of(a.s.T, a.s.S, a.s.L) * a.s.H);
    const size_t e = bf16 ? 2 : 4;
    const bool vec = as_buffer(a.q, a.dk, e, a.s.L) && as_buffer(a.k, a.dk, e, a.s.L) && as_buffer(a.v, a.dv, e, a.s.L) && (!dg || as_buffer(a.x, a.dv, e, a.s.L)) &&
                     out_as_buffer(a.s.H, a.dv, e, a.s.L);
    return with_sizes(bf16, vec, a.dk, a.dv, [&](auto B, auto V, auto K, auto D) {
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(D.value * 4 / walk_columns(K.value, D.value)), 0, stream, a);
            return launched();
        };
        if constexpr (B.value) {
            if (dg) return terms == 3 ? go(walk_kernel<true, K.value, D.value, 3, true, V.value>) : go(walk_kernel<true, K.value, D.value, 2, true, V.value>);
            return terms == 3 ? go(walk_kernel<true, K.value, D.value, 3, false, V.value>) : go(walk_kernel<true, K.value, D.value, 1, false, V.value>);
        } else {
            return dg ? go(walk_kernel<false, K.value, D.value, 1, true, V.value>) : go(walk_kernel<false, K.value, D.value, 1, false, V.value>);
        }
    });
}
// terms: of the log decays' gradient
int back(const BackArgs& a, bool bf16, int terms, bool dg, hipStream_t stream) {
    const unsigned blocks = (unsigned)(slots_of(a.s.T, a.s.S, a.s.L) * a.s.H);
    const size_t e = bf16 ? 2 : 4;
    const bool vec = as_buffer(a.q, a.dk, e, a.s.L) && as_buffer(a.k, a.dk, e, a.s.L) && as_buffer(a.v, a.dv, e, a.s.L) && as_buffer(a.o, a.dv, e, a.s.L) &&
                     out_as_buffer(a.s.H, a.dk, e, a.s.L) && out_as_buffer(a.s.H, a.dv, e, a.s.L);
    return with_sizes(bf16, vec, a.dk, a.dv, [&](auto B, auto V, auto K, auto D) {
        constexpr bool apart = back_apart(K.value, D.value);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(blocks), dim3(back_threads(K.value, D.value)), 0, stream, a);
            return launched();
        };
        if constexpr (apart) {
            int err;
            if constexpr (B.value) err = a.dinitial ? go(back_kernel<true, K.value, D.value, VALUES, 1, 3, false, V.value>) : go(back_kernel<true, K.value, D.value, VALUES, 1, 1, false, V.value>);
            else err = go(back_kernel<false, K.value, D.value, VALUES, 1, 1, false, V.value>);
            if (err) return err;
        }
        constexpr int role = apart ? KEYS : BOTH;
        if constexpr (!B.value) {
            return dg ? go(back_kernel<false, K.value, D.value, role, 1, 1, true, V.value>) : go(back_kernel<false, K.value, D.value, role, 1, 1, false, V.value>);
        } else if constexpr (apart) {
            return !dg ? go(back_kernel<true, K.value, D.value, role, 1, 1, false, V.value>) : terms == 3 ? go(back_kernel<true, K.value, D.value, role, 3, 1, true, V.value>)
                                                                                                : go(back_kernel<true, K.value, D.value, role, 2, 1, true, V.value>);
        } else {
            if (dg)
                return a.dinitial   ? go(back_kernel<true, K.value, D.value, role, 3, 3, true, V.value>)
                       : terms == 3 ? go(back_kernel<true, K.value, D.value, role, 3, 1, true, V.value>)
                                    : go(back_kernel<true, K.value, D.value, role, 2, 1, true, V.value>);
            return a.dinitial ? go(back_kernel<true, K.value, D.value, role, 1, 3, false, V.value>) : go(back_kernel<true, K.value, D.value, role, 1, 1, false, V.value>);
        }
    });
}
// The states at the boundaries: a.bound's, from edge (initial states, or with a.back the gradients of the last ones).
int boundaries(const LocalArgs& a, const float* edge, bool bf16, int terms, hipStream_t stream) {
    const long long n = a.s.T / a.s.L;
    const int elements = a.dk * a.dv;
    const size_t e = bf16 ? 2 : 4;
    const bool vec = as_buffer(a.k, a.dk, e, a.s.L) && as_buffer(a.v, a.dv, e, a.s.L);
    int err = with_sizes(bf16, vec, a.dk, a.dv, [&](auto B, auto V, auto K, auto D) {
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)(n * a.s.H)), dim3(D.value * 4), 0, stream, a);
            return launched();
        };
        if constexpr (B.value)
            return terms == 3   ? go(local_kernel<true, K.value, D.value, 3, V.value>)
                   : terms == 2 ? go(local_kernel<true, K.value, D.value, 2, V.value>)
                                : go(local_kernel<true, K.value, D.value, 1, V.value>);
        else
            return go(local_kernel<false, K.value, D.value, 1, V.value>);
    });
    if (err) return err;
    const bool by_sequence = (long long)a.s.S + 2 <= n, wide = elements % 4 == 0 && aligned(edge, 16);
    const ScanArgs s{a.s, edge, a.bound, a.decay, elements, a.back, by_sequence};
    const unsigned blocks = (unsigned)((by_sequence ? a.s.S + 2 : n) * a.s.H);
    if (wide) hipLaunchKernelGGL((scan_kernel<4>), dim3(blocks, (elements + 1023) / 1024), dim3(256), 0, stream, s);
    else hipLaunchKernelGGL((scan_kernel<1>), dim3(blocks, (elements + 255) / 256), dim3(256), 0, stream, s);
    return launched();
}

}  // namespace
}  // namespace la
}  // namespace nplm

using namespace nplm;
using namespace nplm::la;

extern "C" {

// The rows of a call's blocks, on the host from a host cu: (seq, lo, hi, p0, n, bound) of every place, then of every boundary from 1 on. Returns the number of places.
int64_t nplm_linattn_debug_segments(const int32_t* cu, int32_t S, int64_t T, int32_t L, int64_t* out) {
    const Shape s{cu, nullptr, 0, 0, 0, (int)T, 1, S, L, 0};
    const long long places = slots_of(T, S, L);
    auto put = [&](const Segment& g) {
        for (int64_t v : {(int64_t)g.seq, (int64_t)g.lo, (int64_t)g.hi, (int64_t)g.p0, (int64_t)g.n, (int64_t)g.bound(s)}) *out++ = v;
    };
    for (long long i = 0; i < places; ++i) put(segment_at(s, i));
    for (long long i = 1; i <= T / L; ++i) put(boundary(s, i));
    return places;
}

int32_t nplm_linattn_debug_segment_rows(int64_t T, int32_t H, int32_t S) { return segment_rows(T, H, S); }

size_t nplm_linattn_bounds_bytes(int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act_dtype) {
    if (check_sizes(T, H, S, dk, dv, act_dtype, act_dtype)) return 0;
    const int L = segment_rows(T, H, S);
    return T <= L ? 0 : state_bytes(T, H, L, dk, dv) + decay_bytes(T, H, L);
}

int nplm_linattn_fwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                     const int32_t* cu, const void* log_decay, int64_t g_row, int64_t g_head, float scale, const float* initial, void* o, float* state,
                     void* bounds, size_t bounds_bytes, int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act_dtype, int32_t g_dtype,
                     uint32_t flags, void* stream) {
    if (int e = check_sizes(T, H, S, dk, dv, act_dtype, g_dtype)) return e;
    if (flags & ~(NPLM_LINATTN_REVERSE | NPLM_LINATTN_HEAD_DECAY)) return -NPLM_DWCONV_EFLAGS;
    if (!cu) return -NPLM_DWCONV_ENULL;
    if (!(scale > -INFINITY && scale < INFINITY)) return -NPLM_DWCONV_ESHAPE;
    if (T > 0) {
        for (int e : {check_tensor(q, q_row, q_head, act_dtype), check_tensor(k, k_row, k_head, act_dtype), check_tensor(v, v_row, v_head, act_dtype),
                      check_tensor(log_decay, g_row, g_head, g_dtype)})
            if (e) return e;
        if (!o) return -NPLM_DWCONV_ENULL;
    } else if (!state) {
        return 0;
    }
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16;
    const size_t e = elem(act_dtype);
    if (!aligned(o, dv % 4 == 0 ? 4 * e : e) || !aligned(cu, 4) || !aligned(initial, 4) || !aligned(state, 4)) return -NPLM_DWCONV_EALIGN;
    const int L = segment_rows(T, H, S);
    const size_t need = nplm_linattn_bounds_bytes(T, H, S, dk, dv, act_dtype);
    if (need && (!bounds || !aligned(bounds, 256) || bounds_bytes < need)) return -NPLM_DWCONV_EWORKSPACE;
    const Shape s = shape(cu, log_decay, g_row, g_head, T, H, S, L, g_dtype, flags);
    const Tensor3 tq = tensor(q, q_row, q_head, dk, act_dtype), tk = tensor(k, k_row, k_head, dk, act_dtype), tv = tensor(v, v_row, v_head, dv, act_dtype);
    const States plain{dv, 1};
    float* const bound = need ? (float*)bounds : nullptr;
    // (the gradient of the log decays reads the boundaries, too; a call does not say whether there will be one)
    const int terms = state || g_dtype == NPLM_DWCONV_F32 ? 3 : 2;
    if (need) {
        const LocalArgs a{s, tk, tv, bound, (float*)((char*)bounds + state_bytes(T, H, L, dk, dv)), plain, 1.f, dk, dv, 0};
        if (int err = boundaries(a, initial, bf16, terms, (hipStream_t)stream)) return err;
    }
    const WalkArgs a{s, tq, tk, tv, {}, (char*)o, initial, bound, state, nullptr, plain, scale, dk, dv};
    return walk(a, bf16, state ? 3 : 1, false, (hipStream_t)stream);
}

size_t nplm_linattn_bwd_workspace_bytes(int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv, int32_t act_dtype) {
    if (check_sizes(T, H, S, dk, dv, act_dtype, act_dtype)) return 0;
    // the boundaries' gradients, u [T, H], the segments' sums of one decay a head
    return nplm_linattn_bounds_bytes(T, H, S, dk, dv, act_dtype) + up256((size_t)T * H * sizeof(float)) +
           up256((size_t)slots_of(T, S, segment_rows(T, H, S)) * H * sizeof(double));
}

int nplm_linattn_bwd(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                     const void* dout, int64_t do_row, int64_t do_head, const int32_t* cu, const void* log_decay, int64_t g_row, int64_t g_head, float scale,
                     const float* initial, const float* state, const float* dstate, const void* bounds, size_t bounds_bytes, void* dq, void* dk_out, void* dv_out,
                     void* dlog_decay, float* dinitial, void* workspace, size_t workspace_bytes, int64_t T, int32_t H, int32_t S, int32_t dk, int32_t dv,
                     int32_t act_dtype, int32_t g_dtype, uint32_t flags, void* stream) {
    if (int e = check_sizes(T, H, S, dk, dv, act_dtype, g_dtype)) return e;
    if (flags & ~(NPLM_LINATTN_REVERSE | NPLM_LINATTN_HEAD_DECAY)) return -NPLM_DWCONV_EFLAGS;
    if (!cu) return -NPLM_DWCONV_ENULL;
    if (!(scale > -INFINITY && scale < INFINITY)) return -NPLM_DWCONV_ESHAPE;
    if (T > 0) {
        for (int e : {check_tensor(q, q_row, q_head, act_dtype), check_tensor(k, k_row, k_head, act_dtype), check_tensor(v, v_row, v_head, act_dtype),
                      check_tensor(dout, do_row, do_head, act_dtype), check_tensor(log_decay, g_row, g_head, g_dtype)})
            if (e) return e;
        if (!dq || !dk_out || !dv_out) return -NPLM_DWCONV_ENULL;
    }
    if (dlog_decay && dstate && !state) return -NPLM_DWCONV_ENULL;
    const bool bf16 = act_dtype == NPLM_DWCONV_BF16;
    const size_t e = elem(act_dtype);
    if (!aligned(dq, dk % 4 == 0 ? 4 * e : e) || !aligned(dk_out, dk % 4 == 0 ? 4 * e : e) || !aligned(dv_out, dv % 4 == 0 ? 4 * e : e) || !aligned(cu, 4) ||
        !aligned(dlog_decay, elem(g_dtype)))
        return -NPLM_DWCONV_EALIGN;
    for (const float* t : {initial, state, dstate, (const float*)dinitial})
        if (!aligned(t, 4)) return -NPLM_DWCONV_EALIGN;
    const int L = segment_rows(T, H, S);
    const size_t nb = nplm_linattn_bounds_bytes(T, H, S, dk, dv, act_dtype);
    if (nb && (!bounds || !aligned(bounds, 256) || bounds_bytes < nb)) return -NPLM_DWCONV_EWORKSPACE;
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < nplm_linattn_bwd_workspace_bytes(T, H, S, dk, dv, act_dtype)) return -NPLM_DWCONV_EWORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
    const Shape s = shape(cu, log_decay, g_row, g_head, T, H, S, L, g_dtype, flags);
    const Tensor3 tq = tensor(q, q_row, q_head, dk, act_dtype), tk = tensor(k, k_row, k_head, dk, act_dtype), tv = tensor(v, v_row, v_head, dv, act_dtype),
                  to = tensor(dout, do_row, do_head, dv, act_dtype);
    float* const gbound = nb ? (float*)workspace : nullptr;
    float* const u = (float*)((char*)workspace + nb);
    double* const part = (double*)((char*)u + up256((size_t)T * H * sizeof(float)));
    const bool dg = dlog_decay, one = flags & NPLM_LINATTN_HEAD_DECAY;
    const int dg_terms = !dg ? 1 : g_dtype == NPLM_DWCONV_F32 ? 3 : 2, terms = dinitial ? 3 : dg_terms;
    const float* const bound = nb ? (const float*)bounds : nullptr;
    if (T > 0) {
        if (nb) {
            const LocalArgs a{s, tq, to, gbound, (float*)((char*)workspace + state_bytes(T, H, L, dk, dv)), {dv, 1}, scale, dk, dv, 1};
            if (int err = boundaries(a, dstate, bf16, terms, st)) return err;
        }
        const WalkArgs a{s, to, tv, tk, tq, (char*)dq, initial, bound, nullptr, u, {1, dv}, scale, dv, dk};
        if (int err = walk(a, bf16, dg_terms, dg, st)) return err;
    }
    const BackArgs a{s, tq, tk, tv, to, (char*)dk_out, (char*)dv_out, dstate, gbound, state, bound, initial, u, dinitial, one ? nullptr : (char*)dlog_decay,
                     one && dg ? part : nullptr, g_dtype == NPLM_DWCONV_BF16, scale, dk, dv};
    const long long slots = slots_of(T, S, L);
    if (T > 0 || dinitial || (one && dg)) {
        const int err = back(a, bf16, dg_terms, dg, st);
        if (err) return err;
    }
    if (!one || !dg) return 0;
    hipLaunchKernelGGL(sum_kernel, dim3(H), dim3(256), 0, st, part, slots, H, dlog_decay, (int)(g_dtype == NPLM_DWCONV_BF16));
    return launched();
}

int nplm_linattn_step(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                      const void* log_decay, int64_t g_row, int64_t g_head, float scale, const float* state, float* out_state, const int32_t* slots, void* o,
                      int64_t B, int32_t H, int64_t N, int32_t dk, int32_t dv, int32_t act_dtype, int32_t g_dtype, uint32_t flags, void* stream) {
    if (int e = check_sizes(0, H, 0, dk, dv, act_dtype, g_dtype)) return e;
    if (flags & ~NPLM_LINATTN_HEAD_DECAY) return -NPLM_DWCONV_EFLAGS;
    if (B < 0 || N < 0 || N > INT_MAX || B * H >= kMaxBlocks || B >= kMaxBlocks || (slots ? B > NPLM_LINATTN_MAX_SLOTS : B > N)) return -NPLM_DWCONV_ESHAPE;
    if (!(scale > -INFINITY && scale < INFINITY)) return -NPLM_DWCONV_ESHAPE;
    if (B == 0) return 0;
    for (int e : {check_tensor(q, q_row, q_head, act_dtype), check_tensor(k, k_row, k_head, act_dtype), check_tensor(v, v_row, v_head, act_dtype),
                  check_tensor(log_decay, g_row, g_head, g_dtype)})
        if (e) return e;
    if (!state || !out_state || !o) return -NPLM_DWCONV_ENULL;
    if (!aligned(state, 4) || !aligned(out_state, 4) || !aligned(slots, 4) || !aligned(o, elem(act_dtype))) return -NPLM_DWCONV_EALIGN;
    const size_t ge = elem(g_dtype);
    const StepArgs a{tensor(q, q_row, q_head, dk, act_dtype), tensor(k, k_row, k_head, dk, act_dtype), tensor(v, v_row, v_head, dv, act_dtype),
                     (const char*)log_decay, flags & NPLM_LINATTN_HEAD_DECAY ? 0 : (long long)(g_row * ge), (long long)(g_head * ge), g_dtype == NPLM_DWCONV_BF16,
                     state, out_state, slots, (char*)o, scale, (int)B, H, dk, dv, act_dtype == NPLM_DWCONV_BF16, N};
    // A block has all columns of a state, or 16 of them where there are few states: the chip wants some hundred blocks
    const bool wide = dv % 4 == 0 && aligned(state, 16) && aligned(out_state, 16), few = B * H < 512;
    auto go = [&](auto kernel, int cols) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(B * H), (dv + cols - 1) / cols), dim3(256), 0, (hipStream_t)stream, a);
        return launched();
    };
    // (more than the 256 MB that the last cache holds: the next step finds none of these states in it)
    const bool once = (size_t)B * H * dk * dv * sizeof(float) * (state == out_state ? 1 : 2) > ((size_t)256 << 20);
    if (wide && few) return go(step_kernel<16, 4, false>, 16);
    if (wide && once) return dv > 64 ? go(step_kernel<128, 4, true>, 128) : go(step_kernel<64, 4, true>, 64);
    if (wide) return dv > 64 ? go(step_kernel<128, 4, false>, 128) : go(step_kernel<64, 4, false>, 64);
    return few ? go(step_kernel<16, 1, false>, 16) : go(step_kernel<64, 1, false>, 64);
}

}  // extern "C"
