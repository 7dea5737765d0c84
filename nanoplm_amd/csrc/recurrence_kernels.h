// Kernels of the gated linear recurrence over packed sequences (include/nplm_recurrence.h).
//
// Scan order: row q of the scan is row q of the tensors, or row T - 1 - q with REV; "before" and "after" below are meant in it. A block has
// a slice of 64 * V channels (one lane V of them) and scans chunks of kChunk rows; wave w has the rows [w * RW, (w + 1) * RW) of a chunk.
// Each wave scans its rows as if nothing came before (h, and the product P of the decays up to each row, so that the true state is
// h + P * carry), the waves' last (h, P) meet in the LDS, and every wave folds those before it, in their order, into its carry.
// The backward does the same in the other direction for g (the gradient of h), with h itself restarted from the forward's carries.
#pragma once
#include "dwconv_device.h"

namespace nplm {
namespace rec {

constexpr int kChunk = 64;

struct FwdArgs {
    const char *x, *gates;
    long long xs, gs;                 // row strides in bytes
    const int32_t* cu;
    const void* decay;
    const float* initial;
    char* y;
    float *state, *carries;
    float scale;
    int T, C, S, w_bf16;
};
struct BwdArgs {
    const char *x, *gates, *dy;
    long long xs, gs, ds;
    const int32_t* cu;
    const void* decay;
    const float *initial, *dstate, *carries;
    char *dx, *dgates;
    void* ddecay;
    float *dinitial, *partial;        // partial: ddecay's sums of every chunk, [chunks][C]
    float scale;
    int T, C, S, w_bf16, g_bf16;
};

__device__ __forceinline__ float param_at(const void* p, int i, int bf16) {
    return bf16 ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}
__device__ __forceinline__ float softplus_f32(float v) { return v > 20.f ? v : log1pf(expf(v)); }
// sigmoid(v) / softplus(v): 1 where both vanish
__device__ __forceinline__ float softplus_ratio(float v) {
    const float sp = softplus_f32(v);
    return v < -80.f ? 1.f : 1.f / ((1.f + expf(-v)) * sp);
}

// ---------------------------------------------------------------------------------------------
// The boundaries of cu near a wave's rows. An edge is a place e in [0, T]: between rows e - 1 and e of the tensors. All members are
// wave-uniform and need all lanes; cu's entries lie in the lanes, so an edge costs a ballot. cu is searched 64 entries at a time (two loads up to 4096
// sequences). Indices stay in [0, S] whatever cu holds.
// ---------------------------------------------------------------------------------------------
struct Edges {
    const int32_t* cu;
    uint32_t S, base;     // entries cu[0 .. S]; lane l holds cu[base + l]
    int win;
    bool whole;           // the lanes hold every entry in [lo, hi] and the first one behind

    __device__ __forceinline__ int at(uint32_t i) const { return cu[i < S ? i : S]; }
    // A number n of entries below p, at most 63 short of all of them (all of them, if cu is sorted).
    __device__ __forceinline__ uint32_t search(int p) const {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t lo = 0, hi = S + 1;                      // the answer lies in [lo, hi]
        while (hi - lo > 63) {
            const uint32_t step = (hi - lo + 63) >> 6;
            const uint32_t mine = lo + (lane + 1) * step - 1;
            const uint64_t m = __ballot(mine >= hi || cu[mine < hi ? mine : hi - 1] >= p);
            const uint32_t f = m ? (uint32_t)__builtin_ctzll(m) : 64u;
            lo += f * step;
            const uint32_t end = lo + step - 1;
            hi = f < 64 && end < hi ? end : hi;
            lo = lo < hi ? lo : hi;
        }
        return lo;
    }
    __device__ __forceinline__ void load(uint32_t b) {
        base = b;
        const uint32_t i = b + (threadIdx.x & 63);
        win = i <= S ? cu[i] : 0x7fffffff;
    }
    __device__ __forceinline__ void locate(const int32_t* cu_, int S_, int lo, int hi) {
        cu = cu_;
        S = (uint32_t)S_;
        load(search(lo));
        whole = __builtin_amdgcn_readlane(win, 63) > hi;
    }
    // how many entries lie below p, for p in [lo, hi + 1]
    __device__ __forceinline__ int below(int p) const {
        if (whole) return (int)(base + (uint32_t)__popcll(__ballot(win < p)));
        const uint32_t b = search(p), i = b + (threadIdx.x & 63);
        return (int)(b + (uint32_t)__popcll(__ballot((i <= S ? cu[i] : 0x7fffffff) < p)));
    }
    __device__ __forceinline__ bool hit(int e) const { return whole ? __ballot(win == e) != 0 : below(e + 1) > below(e); }
    // the next edge above e (T: none) or below it (0)
    __device__ __forceinline__ int neighbour(int e, bool up, int T) const {
        const int n = below(up ? e + 1 : e);
        const int v = up ? ((uint32_t)n <= S ? at(n) : T) : n > 0 ? at(n - 1) : 0;
        return __builtin_amdgcn_readfirstlane(v < 0 ? 0 : v > T ? T : v);
    }
    // the sequence that begins / ends at edge e in the scan's order (empty ones left out); outside [0, S): none
    template <bool REV> __device__ __forceinline__ int entered(int e) const { return REV ? below(e) - 1 : below(e + 1) - 1; }
    template <bool REV> __device__ __forceinline__ int left(int e) const { return REV ? below(e + 1) - 1 : below(e) - 1; }
};

// Bit r: an edge lies in front of scan row q0 + r, r = 0 .. N (the edge behind row q0 + N - 1 included).
template <bool REV, int N> __device__ __forceinline__ uint32_t edge_bits(const Edges& ed, int q0, int T) {
    uint32_t bits = 0;
#pragma unroll
    for (int r = 0; r <= N; ++r) {
        const int q = q0 + r;
        if (q <= T && (q == 0 || q == T || ed.hit(REV ? T - q : q))) bits |= 1u << r;
    }
    return bits;
}
template <bool REV> __device__ __forceinline__ int edge_of(int q, int T) { return REV ? T - q : q; }
template <bool REV> __device__ __forceinline__ int row_of(int q, int T) { return REV ? T - 1 - q : q; }

template <int V> __device__ __forceinline__ void load_f32(float (&o)[V], const float* table, int s, int S, int C, int c) {
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = 0.f;
    if (table && (unsigned)s < (unsigned)S) {
        const float* p = table + (size_t)s * C + c;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = p[v];
    }
}
template <int V> __device__ __forceinline__ void store_f32(float* table, int s, int S, int C, int c, const float (&o)[V]) {
    if (table && (unsigned)s < (unsigned)S) {
        float* p = table + (size_t)s * C + c;
#pragma unroll
        for (int v = 0; v < V; ++v) p[v] = o[v];
    }
}

// z = K sigmoid(r) and u = 1 - e^-z: by its series below 1/4 (the first term left out is 5e-8 of it), where 1 - exp would cancel.
// Everything else is made of u without cancellation: a = 1 - u, 1 - a^2 = u (2 - u).
__device__ __forceinline__ void decay_of(float r, float K, float& sr, float& z, float& u) {
    sr = sigmoid_f32(r);
    z = sr * K;
    float s = fmaf(z, -1.f / 720, 1.f / 120);
    s = fmaf(z, s, -1.f / 24);
    s = fmaf(z, s, 1.f / 6);
    s = fmaf(z, s, -0.5f);
    s = fmaf(z, s, 1.f);
    const float far = 1.f - __builtin_amdgcn_exp2f(-1.44269504088896341f * z);
    u = z < 0.25f ? z * s : far;
}

template <int V> struct alignas(8 * V) Pair {
    float A[V], B[V];     // the state behind some rows is A * (state in front) + B
};

// ---------------------------------------------------------------------------------------------
// One scan over many blocks. Each block publishes what its chunk does to a state, A and B of a Pair; the state in front of a chunk is those of
// the chunks before it in the same sequence, folded in order. So that a chunk of a long sequence need not read thousands of them, every
// eighth chunk publishes its group's Pair as well and every 64th the state itself: at most 7 + 7 + 1 are read. What is folded, and in which
// order, goes by the chunk and its sequence alone: results do not depend on which block was faster.
//
// A Pair travels as one 8-byte word a channel, written and read whole at device scope, and says itself whether it is there: A is never negative, and a
// kernel in front of the scan sets the sign bits of all words. Blocks take their chunks by tickets: the blocks with the chunks before a block's
// are running, and each of them publishes a Pair without waiting, a group's Pair waiting for Pairs alone, and a state waiting for
// earlier ones alone: every wait ends.
// ---------------------------------------------------------------------------------------------
constexpr int kGroup = 8, kSuper = 64;       // chunks of a group, chunks of a state

struct Board {
    uint32_t* tickets;                       // one for each slice, 64 bytes apart
    uint64_t *pairs, *groups, *states;       // [chunks][width], [chunks / kGroup][width], [chunks / kSuper][width]
    int chunks, width, slices;               // width: channels, rounded up to whole slices
};
__device__ __forceinline__ void post(uint64_t* at, float A, float B) {
    __hip_atomic_store(at, (uint64_t)__float_as_uint(B) << 32 | (__float_as_uint(A) & 0x7fffffffu), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <int V> __device__ __forceinline__ void post(uint64_t* table, long long row, const Board& b, int c, const float (&A)[V], const float (&B)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) post(table + row * b.width + c + v, A[v], B[v]);
}
template <int V> __device__ __forceinline__ bool missing(const uint64_t (&w)[V]) {
    bool none = false;
#pragma unroll
    for (int v = 0; v < V; ++v) none |= w[v] >> 31 & 1;
    return none;
}
// Folds rows [first, end) of a table, seven at most, into (A, B), which become what they do together; without A, the sequence begins in the first one.
template <int V> __device__ __forceinline__ void fold(const uint64_t* table, int first, int end, bool begins, const Board& b, int c, float (&A)[V], float (&B)[V]) {
    uint64_t w[kGroup - 1][V];
#pragma unroll
    for (int i = 0; i < kGroup - 1; ++i)
        if (first + i < end)
#pragma unroll
            for (int v = 0; v < V; ++v) w[i][v] = peek(table + (long long)(first + i) * b.width + c + v);
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll
    for (int i = 0; i < kGroup - 1; ++i)
        if (first + i < end) {
            while (__ballot(missing<V>(w[i]))) {
                __builtin_amdgcn_s_sleep(2);
#pragma unroll
                for (int v = 0; v < V; ++v) w[i][v] = peek(table + (long long)(first + i) * b.width + c + v);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float a = __uint_as_float((uint32_t)w[i][v]), h = __uint_as_float((uint32_t)(w[i][v] >> 32));
                B[v] = begins && i == 0 ? h : fmaf(a, B[v], h);
                A[v] *= a;
            }
        }
}
// What one wave does for chunk k of a slice: publishes mine (cut: a sequence begins in the chunk, mine.A has no meaning) and returns the state in
// front of the chunk. The sequence of its first row began in chunk ks; ks == k: with that row, there is no state in front.
template <int V> __device__ __forceinline__ void look_back(const Board& b, int k, int ks, const Pair<V>& mine, bool cut, int c, float (&carry)[V]) {
    const int g = k / kGroup, s = k / kSuper;
    const bool ends_group = k % kGroup == kGroup - 1, ends_super = k % kSuper == kSuper - 1, more = k + 1 < b.chunks;
    if (!ends_group && more) post<V>(b.pairs, k, b, c, mine.A, mine.B);
    float A0[V], B0[V];
    const bool in_group = ks >= g * kGroup, in_super = ks >= s * kSuper;
    if (ks < k) fold<V>(b.pairs, in_group ? ks : g * kGroup, k, in_group, b, c, A0, B0);
    if (ends_group && !ends_super && more) {
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = cut ? 0.f : mine.A[v] * A0[v], B[v] = cut ? mine.B[v] : fmaf(mine.A[v], B0[v], mine.B[v]);
        post<V>(b.groups, g, b, c, A, B);
    }
    if (ks < k && in_group) {
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = B0[v];
    } else if (ks < k) {
        float A1[V], B1[V], A2[V], B2[V];
        fold<V>(b.groups, in_super ? ks / kGroup : s * (kSuper / kGroup), g, in_super, b, c, A1, B1);
        if (!in_super) fold<V>(b.states, s - 1, s, true, b, c, A2, B2);
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = fmaf(A0[v], in_super ? B1[v] : fmaf(A1[v], B2[v], B1[v]), B0[v]);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = 0.f;
    }
    if (ends_super && more) {
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 0.f, B[v] = cut ? mine.B[v] : fmaf(mine.A[v], carry[v], mine.B[v]);
        post<V>(b.states, s, b, c, A, B);
    }
}
// The block's ticket in its slice.
__device__ __forceinline__ int take_ticket(const Board& b, int slice, int* lds) {
    if (threadIdx.x == 0) *lds = (int)(atomicAdd(b.tickets + slice * 16, 1u) + 1u);       // (begins at all bits set)
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*lds);
}
// Sets all bits of the board.
__global__ void __launch_bounds__(256) clear_kernel(uint4* at, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) at[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

// What sequences without rows end with: they have no wave.
__device__ __forceinline__ void pass_empty(const int32_t* cu, int S, int C, const float* in, float* out, int first, int step, int c, int n, bool active) {
    if (!out || !active) return;
    for (long long s = first; s < S; s += step)
        if (cu[s + 1] <= cu[s])
            for (int v = 0; v < n; ++v) out[(size_t)s * C + c + v] = in ? in[(size_t)s * C + c + v] : 0.f;
}

// SPLIT: a block scans one chunk of a slice. Else it scans a slice of all rows, a chunk after the other.
template <bool BF16, int V, int NW, bool REV, bool SPLIT>
__global__ void __launch_bounds__(NW * 64) fwd_kernel(const FwdArgs p, const Board board) {
    constexpr int RW = kChunk / NW, E = BF16 ? 2 : 4;
    typedef RowVec<BF16, V> Vec;
    __shared__ Pair<V> agg[2][NW][64];
    __shared__ int cut[2][NW];
    __shared__ float last[2][64 * V];
    __shared__ int ticket;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = SPLIT ? blockIdx.x % board.slices : blockIdx.x;
    const int c0 = (slice * 64 + lane) * V;
    const bool active = c0 < p.C;
    const int c = active ? c0 : p.C - V;
    float K[V];
#pragma unroll
    for (int v = 0; v < V; ++v) K[v] = p.scale * softplus_f32(param_at(p.decay, c + v, p.w_bf16));
    const int nchunks = (p.T + kChunk - 1) / kChunk;
    const int k0 = SPLIT ? take_ticket(board, slice, &ticket) : 0, k1 = SPLIT ? k0 + 1 : nchunks;
    pass_empty(p.cu, p.S, p.C, p.initial, p.state, k0 * NW + wave, SPLIT ? nchunks * NW : NW, c, V, active);
    if (!SPLIT && threadIdx.x < 64)
#pragma unroll
        for (int v = 0; v < V; ++v) last[1][lane * V + v] = 0.f;

    for (int k = k0; k < k1; ++k) {
        const int q0 = k * kChunk + wave * RW, par = k & 1;
        const int e0 = edge_of<REV>(q0, p.T), e1 = edge_of<REV>(q0 + RW, p.T);
        float h[RW][V], P[RW][V];
        Vec xv[RW], rv[RW], iv[RW];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            const int q = q0 + r < p.T ? q0 + r : p.T - 1;
            const size_t t = (size_t)row_of<REV>(q, p.T);
            xv[r].load(p.x + t * p.xs + (uint32_t)c * E);
            rv[r].load(p.gates + t * p.gs + (uint32_t)c * E);
            iv[r].load(p.gates + t * p.gs + (size_t)p.C * E + (uint32_t)c * E);
        }
        Edges ed;
        ed.locate(p.cu, p.S, REV ? e1 : e0, REV ? e0 : e1);
        const uint32_t edges = edge_bits<REV, RW>(ed, q0, p.T);
        const uint32_t starts = edges & ((1u << RW) - 1);
        const int fs = starts ? __builtin_ctz(starts) : RW;        // rows in front of it take the carry
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float x[V], rg[V], ig[V], h0[V];
            xv[r].to_f32(x);
            rv[r].to_f32(rg);
            iv[r].to_f32(ig);
            const bool real = q0 + r < p.T, start = starts >> r & 1;
            if (start) load_f32<V>(h0, p.initial, ed.template entered<REV>(edge_of<REV>(q0 + r, p.T)), p.S, p.C, c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float sr, z, u;
                decay_of(rg[v], K[v], sr, z, u);
                const float beta = __builtin_amdgcn_sqrtf(fmaf(-u, u, u + u));
                float a = 1.f - u, b = beta * sigmoid_f32(ig[v]) * x[v];
                if (!real) a = 1.f, b = 0.f;
                h[r][v] = start ? fmaf(a, h0[v], b) : r ? fmaf(a, h[r - 1][v], b) : b;
                P[r][v] = r ? a * P[r - 1][v] : a;
            }
        }
        Pair<V> mine;
#pragma unroll
        for (int v = 0; v < V; ++v) mine.A[v] = P[RW - 1][v], mine.B[v] = h[RW - 1][v];
        agg[par][wave][lane] = mine;
        if (lane == 0) cut[par][wave] = fs < RW;
        __syncthreads();
        if constexpr (SPLIT) {
            if (wave == 0) {
                Pair<V> all = mine;
                bool any = fs < RW;
                for (int w = 1; w < NW; ++w) {
                    const Pair<V> f = agg[par][w][lane];
                    const bool whole = cut[par][w] == 0;
                    any |= !whole;
#pragma unroll
                    for (int v = 0; v < V; ++v) all.A[v] *= f.A[v], all.B[v] = whole ? fmaf(f.A[v], all.B[v], f.B[v]) : f.B[v];
                }
                const int qs = starts & 1 ? q0 : REV ? p.T - ed.neighbour(e0, true, p.T) : ed.neighbour(e0, false, p.T);
                float front[V];
                look_back<V>(board, k, starts & 1 ? k : (qs < q0 ? qs : q0 - 1) / kChunk, all, any, c0, front);
#pragma unroll
                for (int v = 0; v < V; ++v) last[1 - par][lane * V + v] = front[v];
            }
            __syncthreads();
        }
        float carry[V];
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = last[1 - par][lane * V + v];
        if (wave == 0 && p.carries && active)
#pragma unroll
            for (int v = 0; v < V; ++v) p.carries[(size_t)k * p.C + c + v] = carry[v];
        for (int w = 0; w < wave; ++w) {
            const Pair<V> f = agg[par][w][lane];
            const bool whole = cut[par][w] == 0;
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = whole ? fmaf(f.A[v], carry[v], f.B[v]) : f.B[v];
        }
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            if (r < fs)
#pragma unroll
                for (int v = 0; v < V; ++v) h[r][v] = fmaf(P[r][v], carry[v], h[r][v]);
            int done = -1;                                          // (found with all lanes)
            if (p.state && q0 + r < p.T && (edges >> (r + 1) & 1)) done = ed.template left<REV>(edge_of<REV>(q0 + r + 1, p.T));
            if (active && q0 + r < p.T) {
                Vec o;
                o.from_f32(h[r]);
                o.store(p.y + ((size_t)row_of<REV>(q0 + r, p.T) * p.C + c) * E);
                store_f32<V>(p.state, done, p.S, p.C, c, h[r]);
            }
        }
        if (!SPLIT && wave == NW - 1)
#pragma unroll
            for (int v = 0; v < V; ++v) last[par][lane * V + v] = h[RW - 1][v];
    }
}

// The backward, chunks from the scan's end to its beginning. gamma is what comes back to a row's h from behind it:
// g_t = dy_t + gamma_t, gamma_{t-1} = a_t g_t.
template <bool BF16, int V, int NW, bool REV, bool SPLIT>
__global__ void __launch_bounds__(NW * 64) bwd_kernel(const BwdArgs p, const Board board) {
    constexpr int RW = kChunk / NW, E = BF16 ? 2 : 4;
    typedef RowVec<BF16, V> Vec;
    __shared__ Pair<V> fwd[2][NW][64], bwd[2][NW][64];
    __shared__ int cut[2][NW];
    __shared__ float first[2][64 * V];
    __shared__ int ticket;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = SPLIT ? blockIdx.x % board.slices : blockIdx.x;
    const int c0 = (slice * 64 + lane) * V;
    const bool active = c0 < p.C;
    const int c = active ? c0 : p.C - V;
    float K[V];
    double total[V];
#pragma unroll
    for (int v = 0; v < V; ++v) K[v] = p.scale * softplus_f32(param_at(p.decay, c + v, p.w_bf16)), total[v] = 0;
    const int nchunks = (p.T + kChunk - 1) / kChunk;
    const int k0 = SPLIT ? nchunks - 1 - take_ticket(board, slice, &ticket) : nchunks - 1, k1 = SPLIT ? k0 : 0;
    pass_empty(p.cu, p.S, p.C, p.dstate, p.dinitial, (SPLIT ? k0 * NW : 0) + wave, SPLIT ? nchunks * NW : NW, c, V, active);
    if (!SPLIT && threadIdx.x < 64)
#pragma unroll
        for (int v = 0; v < V; ++v) first[nchunks & 1][lane * V + v] = 0.f;
    for (int k = k0; k >= k1; --k) {
        const int q0 = k * kChunk + wave * RW, par = k & 1;
        const int e0 = edge_of<REV>(q0, p.T), e1 = edge_of<REV>(q0 + RW, p.T);
        Vec xv[RW], rv[RW], iv[RW], dv[RW];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            const int q = q0 + r < p.T ? q0 + r : p.T - 1;
            const size_t t = (size_t)row_of<REV>(q, p.T);
            xv[r].load(p.x + t * p.xs + (uint32_t)c * E);
            rv[r].load(p.gates + t * p.gs + (uint32_t)c * E);
            iv[r].load(p.gates + t * p.gs + (size_t)p.C * E + (uint32_t)c * E);
            dv[r].load(p.dy + t * p.ds + (uint32_t)c * E);
        }
        float carry[V];
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = p.carries[(size_t)k * p.C + c + v];
        Edges ed;
        ed.locate(p.cu, p.S, REV ? e1 : e0, REV ? e0 : e1);
        const uint32_t edges = edge_bits<REV, RW>(ed, q0, p.T);
        const uint32_t starts = edges & ((1u << RW) - 1);
        const int fs = starts ? __builtin_ctz(starts) : RW;           // rows in front of it continue what came before the wave
        const int ls = starts ? 31 - __builtin_clz(starts) : 0;       // rows from it on reach what comes behind the wave

        // dx = g p1, di = g p2, dr = m nr with m = g (U + W carry), the gradient of z times z: every gradient is linear in g
        float p1[RW][V], p2[RW][V], nr[RW][V], U[RW][V], W[RW][V], g[RW][V], Q[RW][V], a[RW][V];
        float h[V], P[V];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float x[V], rg[V], ig[V], h0[V];
            xv[r].to_f32(x);
            rv[r].to_f32(rg);
            iv[r].to_f32(ig);
            dv[r].to_f32(g[r]);
            const bool real = q0 + r < p.T, start = starts >> r & 1;
            if (start) load_f32<V>(h0, p.initial, ed.template entered<REV>(edge_of<REV>(q0 + r, p.T)), p.S, p.C, c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float sr, z, u;
                decay_of(rg[v], K[v], sr, z, u);
                const float beta2 = fmaf(-u, u, u + u);
                const float ib = __builtin_amdgcn_rsqf(fmaxf(beta2, 1e-37f));
                const float si = sigmoid_f32(ig[v]);
                a[r][v] = real ? 1.f - u : 1.f;
                p1[r][v] = beta2 * ib * si;
                const float b = real ? p1[r][v] * x[v] : 0.f;
                p2[r][v] = b * (1.f - si);
                nr[r][v] = 1.f - sr;
                const float ai = a[r][v] * ib, za = z * a[r][v];
                const float before = start ? h0[v] : r ? h[v] : 0.f, scaled = start ? 0.f : r ? P[v] : 1.f;
                U[r][v] = real ? z * (b * ai * ai) - za * before : 0.f;
                W[r][v] = real ? -za * scaled : 0.f;
                h[v] = fmaf(a[r][v], before, b);
                P[v] = a[r][v] * scaled;
                if (!real) g[r][v] = 0.f;
            }
        }
#pragma unroll
        for (int r = RW - 1; r >= 0; --r) {
            if (edges >> (r + 1) & 1) {
                if (p.dstate && q0 + r < p.T) {
                    float d[V];
                    load_f32<V>(d, p.dstate, ed.template left<REV>(edge_of<REV>(q0 + r + 1, p.T)), p.S, p.C, c);
#pragma unroll
                    for (int v = 0; v < V; ++v) g[r][v] += d[v];
                }
            } else if (r < RW - 1) {
#pragma unroll
                for (int v = 0; v < V; ++v) g[r][v] = fmaf(a[r + 1][v], g[r + 1][v], g[r][v]);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) Q[r][v] = r < RW - 1 ? a[r + 1][v] * Q[r + 1][v] : 1.f;
        }
        Pair<V> f, b;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            f.A[v] = P[v];
            f.B[v] = h[v];
            b.A[v] = starts & 1 ? 0.f : a[0][v] * Q[0][v];
            b.B[v] = starts & 1 ? 0.f : a[0][v] * g[0][v];
        }
        fwd[par][wave][lane] = f;
        bwd[par][wave][lane] = b;
        if (lane == 0) cut[par][wave] = fs < RW;
        __syncthreads();
        for (int w = 0; w < wave; ++w) {
            const Pair<V> f = fwd[par][w][lane];
            const bool whole = cut[par][w] == 0;
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = whole ? fmaf(f.A[v], carry[v], f.B[v]) : f.B[v];
        }
        if constexpr (SPLIT) {
            if (wave == NW - 1) {
                Pair<V> all = b;
                bool any = fs < RW;
                for (int w = NW - 2; w >= 0; --w) {
                    const Pair<V> f = bwd[par][w][lane];
                    const bool whole = cut[par][w] == 0;
                    any |= !whole;
#pragma unroll
                    for (int v = 0; v < V; ++v) all.A[v] *= f.A[v], all.B[v] = whole ? fmaf(f.A[v], all.B[v], f.B[v]) : f.B[v];
                }
                // the chunk that the sequence of the last row ends in
                const bool ended = edges >> RW & 1 || q0 + RW >= p.T;
                const int qe = ended ? q0 + RW : REV ? p.T - ed.neighbour(e1, false, p.T) : ed.neighbour(e1, true, p.T);
                const int ke = ended ? k : (qe > q0 + RW ? qe - 1 : q0 + RW) / kChunk;
                float behind[V];
                look_back<V>(board, nchunks - 1 - k, nchunks - 1 - ke, all, any, c0, behind);
#pragma unroll
                for (int v = 0; v < V; ++v) first[1 - par][lane * V + v] = behind[v];
            }
            __syncthreads();
        }
        float gamma[V];
#pragma unroll
        for (int v = 0; v < V; ++v) gamma[v] = first[1 - par][lane * V + v];
        for (int w = NW - 1; w > wave; --w) {
            const Pair<V> f = bwd[par][w][lane];
            const bool whole = cut[par][w] == 0;
#pragma unroll
            for (int v = 0; v < V; ++v) gamma[v] = whole ? fmaf(f.A[v], gamma[v], f.B[v]) : f.B[v];
        }
        const bool into = !(edges >> RW & 1);         // something of the wave's last sequence comes behind it
        float g0[V], sum[V];
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] = 0.f;
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float dx[V], dr[V], di[V], gr[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gr[v] = into && r >= ls ? fmaf(Q[r][v], gamma[v], g[r][v]) : g[r][v];
                const float m = gr[v] * (r < fs ? fmaf(W[r][v], carry[v], U[r][v]) : U[r][v]);
                sum[v] += m;
                dx[v] = gr[v] * p1[r][v];
                dr[v] = m * nr[r][v];
                di[v] = gr[v] * p2[r][v];
                if (r == 0) g0[v] = gr[v];
            }
            int begun = -1;
            if (p.dinitial && q0 + r < p.T && (starts >> r & 1)) begun = ed.template entered<REV>(edge_of<REV>(q0 + r, p.T));
            if (active && q0 + r < p.T) {
                const size_t t = (size_t)row_of<REV>(q0 + r, p.T);
                Vec o;
                o.from_f32(dx);
                o.store(p.dx + (t * p.C + c) * E);
                o.from_f32(dr);
                o.store(p.dgates + (2 * t * p.C + c) * E);
                o.from_f32(di);
                o.store(p.dgates + ((2 * t + 1) * p.C + c) * E);
                if (begun >= 0) {
                    float d[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) d[v] = a[r][v] * gr[v];
                    store_f32<V>(p.dinitial, begun, p.S, p.C, c, d);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) total[v] += sum[v];
        if (!SPLIT && wave == 0)
#pragma unroll
            for (int v = 0; v < V; ++v) first[par][lane * V + v] = starts & 1 ? 0.f : a[0][v] * g0[v];
    }
    __shared__ double sums[NW][64 * V];
#pragma unroll
    for (int v = 0; v < V; ++v) sums[wave][lane * V + v] = total[v];
    __syncthreads();
    if (wave == 0 && active) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            double d = 0;
            for (int w = 0; w < NW; ++w) d += sums[w][lane * V + v];
            if (SPLIT) {
                p.partial[(size_t)k0 * p.C + c + v] = (float)d;
                continue;
            }
            const float o = (float)(d * softplus_ratio(param_at(p.decay, c + v, p.w_bf16)));
            if (p.g_bf16) ((uint16_t*)p.ddecay)[c + v] = f32_to_bf16(o);
            else ((float*)p.ddecay)[c + v] = o;
        }
    }
}

// Adds up the chunks' sums for ddecay in fp64. A block has 16 channels and 64 groups of lanes that each take every 64th chunk.
__global__ void __launch_bounds__(1024) sum_kernel(const float* __restrict__ partial, const void* decay, void* ddecay, int chunks, int C, int w_bf16, int g_bf16) {
    __shared__ double part[64][16];
    const int j = threadIdx.x / 16, i = threadIdx.x % 16, c = blockIdx.x * 16 + i;
    double s = 0;
    if (c < C) {
        int k = j;
        for (; k + 7 * 64 < chunks; k += 8 * 64) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = partial[(size_t)(k + u * 64) * C + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; k < chunks; k += 64) s += partial[(size_t)k * C + c];
    }
    part[j][i] = s;
    __syncthreads();
    if (j || c >= C) return;
    s = 0;
#pragma unroll 8
    for (int u = 0; u < 64; ++u) s += part[u][i];
    const float o = (float)(s * softplus_ratio(param_at(decay, c, w_bf16)));
    if (g_bf16) ((uint16_t*)ddecay)[c] = f32_to_bf16(o);
    else ((float*)ddecay)[c] = o;
}

// One token of each of B sequences. A block has a row and 256 * V channels of it. The row that names a slot first also computes the later
// rows that name it, in their order; they do nothing. To find them out, a block reads all B slots.
struct StepArgs {
    const char *x, *gates;
    long long xs, gs;
    const void* decay;
    const float* state;
    float* out_state;
    const int32_t* slots;
    char* y;
    float scale;
    long long N;
    int B, C, w_bf16;
};
template <bool BF16>
__global__ void __launch_bounds__(256) step_kernel(const StepArgs p) {
    constexpr int E = BF16 ? 2 : 4;
    typedef RowVec<BF16, 1> Vec;
    const int b = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x;
    const bool active = c < p.C;
    const long long slot = p.slots ? p.slots[b] : b;
    if (slot < 0 || slot >= p.N) {
        Vec o;
        const float zero[1] = {0.f};
        o.from_f32(zero);
        if (active) o.store(p.y + ((size_t)b * p.C + c) * E);
        return;
    }
    const int cc = active ? c : p.C - 1;
    float h = p.state[(size_t)slot * p.C + cc];
    Vec xv, rv, iv;
    auto load = [&](int j) {
        xv.load(p.x + j * p.xs + (size_t)cc * E);
        rv.load(p.gates + j * p.gs + (size_t)cc * E);
        iv.load(p.gates + j * p.gs + ((size_t)p.C + cc) * E);
    };
    load(b);
    const float K = p.scale * softplus_f32(param_at(p.decay, cc, p.w_bf16));
    bool more = false;
    if (p.slots) {
        bool before = false, behind = false;
        for (int j = threadIdx.x; j < p.B; j += 256)
            if (p.slots[j] == slot) before |= j < b, behind |= j > b;
        if (__syncthreads_or(before)) return;
        more = __syncthreads_or(behind);
    }
    for (int j = b;;) {
        float x[1], r[1], i[1], sr, z, u;
        xv.to_f32(x);
        rv.to_f32(r);
        iv.to_f32(i);
        decay_of(r[0], K, sr, z, u);
        h = fmaf(1.f - u, h, __builtin_amdgcn_sqrtf(fmaf(-u, u, u + u)) * sigmoid_f32(i[0]) * x[0]);
        const float o[1] = {h};
        xv.from_f32(o);
        if (active) xv.store(p.y + ((size_t)j * p.C + c) * E);
        if (!more) break;
        for (++j; j < p.B && p.slots[j] != slot; ++j) {}
        if (j == p.B) break;
        load(j);
    }
    if (active) p.out_state[(size_t)slot * p.C + c] = h;
}

}  // namespace rec
}  // namespace nplm
