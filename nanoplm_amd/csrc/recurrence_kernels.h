// Kernels of the gated linear recurrence over packed sequences (include/nplm_recurrence.h).
//
// Scan order: row q of the scan is row q of the tensors, or row T - 1 - q with REV; "before" and "behind" below are meant in it. A block has
// a slice of 64 * V channels (one lane V of them) and scans chunks of rows; wave w has the rows [w * RW, (w + 1) * RW) of a chunk.
// Each wave scans its rows as if nothing came before (h, and the product P of the decays up to each row, so that the true state is
// h + P * carry), the waves' last (h, P) meet in the LDS, and every wave folds those before it, in their order, into its carry.
// The backward does the same in the other direction for g (the gradient of h), with h itself restarted from the forward's carries.
#pragma once
#include <type_traits>

#include "dwconv_device.h"

// Products and sums are fused where it says fmaf and nowhere else: all variants of a kernel give the same bits.
#pragma clang fp contract(off)

namespace nplm {
namespace rec {

constexpr int kCarryRows = 32;             // rows between the states that the forward leaves

// Waves of a block, the rows of a chunk that each of them has, waves that a SIMD's registers hold. The look-back's round trips and words are paid once a chunk
// and the boundaries once a wave, so that chunks are as long as registers allow; T=131072, C=1024, bf16, packed, us (before its loads went past the caches):
// forward, waves x rows: 8 x 8 335, 4 x 16 283, 8 x 16 254, 12 x 16 319 (one block a CU), 16 x 16 294; backward 4 x 8 600 (3 blocks a CU), 8 x 8 614,
// 12 x 8 605, 4 x 16 540.
struct Shape {
    int waves, rows, eu;
    constexpr int chunk() const { return waves * rows; }
};
constexpr Shape fwd_shape(bool bf16) { return bf16 ? Shape{8, 16, 4} : Shape{8, 8, 4}; }
constexpr Shape bwd_shape(bool bf16) { return bf16 ? Shape{4, 16, 2} : Shape{4, 8, 3}; }

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
// The boundaries of cu around N rows of a wave. An edge is a place e in [0, T]: between rows e - 1 and e of the tensors. All of it is scalar, and cu is read
// by scalar loads, which do not queue behind the rows that the wave has asked for: the search is over before they are there. Indices stay in [0, S]
// whatever cu holds.
// ---------------------------------------------------------------------------------------------
template <bool REV, int N> struct Edges {
    ScalarCu cu;
    int S, T, q0;
    uint32_t bits;        // bit r: an edge in front of the wave's row r of the scan, r = 0 .. N

    // how many entries lie below p
    __device__ __forceinline__ int below(int p) const {
        uint32_t lo = 0, hi = (uint32_t)S + 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (cu_at(cu, (int)mid) < p) lo = mid + 1; else hi = mid;
        }
        return (int)lo;
    }
    // Rows first .. first + N - 1 of the scan.
    __device__ __forceinline__ void locate(const int32_t* cu_, int S_, int first, int T_) {
        cu.p = cu_;
        S = S_;
        T = T_;
        q0 = first;
        const int lo = REV ? T - q0 - N : q0, hi = lo + N;
        bits = q0 == 0 ? 1u : 0u;
        int i = below(lo);
        while ((uint32_t)i <= (uint32_t)S) {
            const int e = cu_at(cu, i);
            if (e > hi) break;
            if (e >= lo) bits |= 1u << (REV ? T - e - q0 : e - q0);
            ++i;
            if ((uint32_t)i <= (uint32_t)S && cu_at(cu, i) == e) {     // a run of empty sequences
                const int behind = below(e + 1);
                i = behind > i ? behind : i + 1;
            }
        }
        const int n = T - q0;                             // rows that there are; the edge behind the last one always is
        if (n <= N) bits = n < 0 ? 0u : (bits & ((1u << n) - 1)) | 1u << n;
    }
    __device__ __forceinline__ int edge(int r) const { return REV ? T - q0 - r : q0 + r; }
    // the sequence that begins in front of row r / ends in front of row r, in the scan's order (empty ones left out); outside [0, S): none
    __device__ __forceinline__ int entered(int r) const { return below(edge(r) + (REV ? 0 : 1)) - 1; }
    __device__ __forceinline__ int left(int r) const { return below(edge(r) + (REV ? 1 : 0)) - 1; }
    // the place q in the scan of the next edge before row r's / behind it, for an r whose own place is no edge
    __device__ __forceinline__ int before(int r) const { return place(r, true); }
    __device__ __forceinline__ int behind(int r) const { return place(r, false); }
    __device__ __forceinline__ int place(int r, bool back) const {
        const int n = below(edge(r));                     // (none is at the edge)
        const bool up = REV == back;                      // towards higher rows of the tensors
        const uint32_t i = up ? (uint32_t)n : (uint32_t)n - 1;
        int e = up ? T : 0;
        if (i <= (uint32_t)S) e = cu_at(cu, (int)i);
        e = e < 0 ? 0 : e > T ? T : e;
        return REV ? T - e : e;
    }
};

// Where a wave's rows lie. Buffer addressing: a descriptor at the first of the rows in memory, a scalar offset for the row, a lane's offset for its
// channels, so that addresses take no vector ALU work. Rows behind the last one of the tensors read the last one and are not stored.
template <bool REV, int N> struct Rows {
    int t, n, most;       // first row in memory, rows that there are (of N; may be negative), index of the last row that may be touched
    __device__ __forceinline__ void set(int q0, int T) {
        n = T - q0 < N ? T - q0 : N;
        most = n > 0 ? n - 1 : 0;
        const int q = q0 < T ? q0 : T - 1;
        t = REV ? T - 1 - q - most : q;
    }
    __device__ __forceinline__ rsrc_t at(const char* p, long long stride) const { return make_rsrc(p + (long long)t * stride, 0x7fffffffu); }
    __device__ __forceinline__ int off(int r, int stride) const {
        const int j = r < most ? r : most;
        return (REV ? most - j : j) * stride;
    }
};

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

// Keeps the compiler from widening all rows of a wave in front of the branch that all of its ways widen them behind: that took the registers of a block.
template <int WAY> __device__ __forceinline__ void stay(uint32_t& d) {
    if constexpr (WAY == 0) asm volatile("; rows with an edge" : "+v"(d));
    else if constexpr (WAY == 1) asm volatile("; plain rows" : "+v"(d));
    else if constexpr (WAY == 2) asm volatile("; plain rows of slow decays" : "+v"(d));
    else asm volatile("; plain rows again" : "+v"(d));
}
template <int WAY, int V> __device__ __forceinline__ void stay(RowVec<true, V>& r) {
    if constexpr (V == 1) {
        uint32_t h = r.h;
        stay<WAY>(h);
        r.h = (uint16_t)h;
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) stay<WAY>(r.d[i]);
    }
}
template <int WAY, int V> __device__ __forceinline__ void stay(RowVec<false, V>&) {}

// z = K sigmoid(r) and u = 1 - e^-z: by its series below 1/4 (the first term left out is 5e-8 of it), where 1 - exp would cancel.
// Everything else is made of u without cancellation: 1 - a^2 = u (2 - u); a = 1 - u where the series holds, else the exponential itself, which keeps its digits
// where it is small. NEAR: K is below 1/4, and so is every z.
template <bool NEAR> __device__ __forceinline__ void decay_of(float r, float K, float& sr, float& z, float& u, float& a) {
    sr = sigmoid_f32(r);
    z = sr * K;
    float s = fmaf(z, -1.f / 720, 1.f / 120);
    s = fmaf(z, s, -1.f / 24);
    s = fmaf(z, s, 1.f / 6);
    s = fmaf(z, s, -0.5f);
    s = fmaf(z, s, 1.f);
    u = z * s;
    a = 1.f - u;
    if constexpr (!NEAR) {
        const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * z);
        u = z < 0.25f ? u : 1.f - e;
        a = z < 0.25f ? a : e;
    }
}
// Whether no channel of the wave forgets more than 22 % a token (decays in use are slower by far): its rows without an edge then take a sixth less of
// the vector ALU's time in the forward.
template <int V> __device__ __forceinline__ bool all_near(const float (&K)[V]) {
    bool far = false;
#pragma unroll
    for (int v = 0; v < V; ++v) far |= !(K[v] < 0.25f);
    return __ballot(far) == 0;
}

template <int V> struct alignas(8 * V) Pair {
    float A[V], B[V];     // the state behind some rows is A * (state in front) + B
};
// A, a product of many decays, is never 0, also where that is what is left of it in fp32: an infinite state in front then stays infinite, as it does row by row.
// (Denormals count. Here and not where A meets the state, which is what other blocks wait for.)
__device__ __forceinline__ float left_of(float A) { return fmaxf(A, 0x1p-149f); }

// ---------------------------------------------------------------------------------------------
// One scan over many blocks. Each block publishes what its chunk does to a state, A and B of a Pair; the state in front of a chunk is made of those of
// the chunks before it in the same sequence, in order. So that a chunk of a long sequence need not read thousands of them, every
// eighth chunk publishes its group's Pair as well and every 64th the state itself: at most 7 + 7 + 1 are read, by one wave of the block. What is
// folded, and in which order, goes by the chunk and its sequence alone: results do not depend on which block was faster.
//
// A Pair travels as one 8-byte word a channel, written and read whole at device scope, and says itself whether it is there: A is never negative, and a
// kernel in front of the scan sets the sign bits of all words. Blocks take their chunks by tickets, in the scan's order: of the chunks that are not finished, the
// first one's block is running, and all that it waits for is there. So every wait ends.
// ---------------------------------------------------------------------------------------------
constexpr int kGroup = 8, kSuper = 64;       // chunks of a group, chunks of a state

struct Board {
    uint32_t* tickets;                       // one for each slice, 64 bytes apart
    uint64_t *pairs, *groups, *states;       // [chunks][width], [chunks / kGroup][width], [chunks / kSuper][width]
    float* K;                                // scale * softplus(decay)
    int chunks, width, slices;               // width: channels, rounded up to whole slices
};
template <int V> __device__ __forceinline__ void post(uint64_t* table, int row, const Board& b, int c, const float (&A)[V], const float (&B)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v)
        __hip_atomic_store(table + (long long)row * b.width + c + v, (uint64_t)__float_as_uint(B[v]) << 32 | (__float_as_uint(A[v]) & 0x7fffffffu),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <int V> __device__ __forceinline__ void peek(uint64_t (&w)[V], const uint64_t* table, int row, const Board& b, int c) {
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = __hip_atomic_load(table + (long long)row * b.width + c + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int V> __device__ __forceinline__ bool missing(const uint64_t (&w)[V]) {
    bool none = false;
#pragma unroll
    for (int v = 0; v < V; ++v) none |= w[v] >> 31 & 1;
    return none;
}
// Folds rows [first, end) of a table into (A, B), which become what they do together; with begins, the sequence begins in the first one. Four of them are
// asked for at a time.
template <int V> __device__ __forceinline__ void fold(const uint64_t* table, int first, int end, bool begins, const Board& b, int c, float (&A)[V], float (&B)[V]) {
    constexpr int AT_ONCE = 4;
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
    for (; first < end; first += AT_ONCE) {
        uint64_t w[AT_ONCE][V];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (first + i < end) peek<V>(w[i], table, first + i, b, c);
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (first + i < end) {
                while (__ballot(missing<V>(w[i]))) {
                    __builtin_amdgcn_s_sleep(16);             // (words read too often fill the fabric)
                    peek<V>(w[i], table, first + i, b, c);
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float a = __uint_as_float((uint32_t)w[i][v]), h = __uint_as_float((uint32_t)(w[i][v] >> 32));
                    B[v] = begins ? h : fmaf(a, B[v], h);
                    A[v] *= a;
                }
                begins = false;
            }
    }
}
// What one wave does for chunk k of a slice: publishes mine (cut: a sequence begins in the chunk, mine.A has no meaning) and returns the state in
// front of the chunk. The sequence of its first row began in chunk ks; ks == k: with that row, there is no state in front.
template <int V> __device__ __forceinline__ void look_back(const Board& b, int k, int ks, const Pair<V>& mine, bool cut, int c, float (&carry)[V]) {
    const int g = k / kGroup, s = k / kSuper;
    const bool ends_group = k % kGroup == kGroup - 1, ends_super = k % kSuper == kSuper - 1, more = k + 1 < b.chunks;
    if (!ends_group && more) post<V>(b.pairs, k, b, c, mine.A, mine.B);
    float A0[V] = {}, B0[V] = {};          // (nothing in front, also where no cut says so: a sequence may fill a chunk from end to end)
    const bool in_group = ks >= g * kGroup, in_super = ks >= s * kSuper;
    if (ks < k) fold<V>(b.pairs, in_group ? ks : g * kGroup, k, in_group, b, c, A0, B0);
    if (ends_group && !ends_super && more) {
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = cut ? 0.f : left_of(mine.A[v] * A0[v]), B[v] = cut ? mine.B[v] : fmaf(mine.A[v], B0[v], mine.B[v]);
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
        for (int v = 0; v < V; ++v) carry[v] = fmaf(left_of(A0[v]), in_super ? B1[v] : fmaf(left_of(A1[v]), B2[v], B1[v]), B0[v]);
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
// The block's ticket in its slice (they begin at all bits set).
__device__ __forceinline__ int take_ticket(const Board& b, int slice, int* lds) {
    if (threadIdx.x == 0) *lds = (int)(atomicAdd(b.tickets + slice * 16, 1u) + 1u);
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*lds);
}
// In front of a scan: sets all bits of the board, n times 16 bytes, and forms K.
__global__ void __launch_bounds__(256) prepare_kernel(uint4* at, long long n, float* K, const void* decay, float scale, int C, int w_bf16) {
    const long long first = (long long)blockIdx.x * 256 + threadIdx.x, step = (long long)gridDim.x * 256;
    for (long long i = first; i < n; i += step) at[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
    for (long long c = first; c < C; c += step) K[c] = scale * softplus_f32(param_at(decay, c, w_bf16));
}

// What sequences without rows end with: they have no wave.
__device__ __forceinline__ void pass_empty(const int32_t* cu, int S, int C, const float* in, float* out, int first, int step, int c, int n, bool active) {
    if (!out || !active) return;
    for (long long s = first; s < S; s += step)
        if (cu[s + 1] <= cu[s])
            for (int v = 0; v < n; ++v) out[(size_t)s * C + c + v] = in ? in[(size_t)s * C + c + v] : 0.f;
}

// Bound by memory and by what its waves wait for before and behind the look-back: T=131072, C=1024, bf16 246 us (4.4 TB/s; a copy of 256 MiB here reaches 5.6, with nt hints 6.2), fp32
// T=32768, C=768 86 us (4.7), one sequence of bf16 T=65536, C=2048 238 us (4.5); the vector ALU is busy for half of it.
// A block scans one chunk of a slice. SPLIT: of several. Else there is one chunk, nothing to look back at and no kernel in front (T=64, C=1024, bf16: forward 10
// and 13.5 us, backward 13 and 19; one block that goes on to a second chunk is slower than two already in the backward, and at 512 rows 27 and 61 us
// against 13 and 19).
template <bool BF16, int V, bool REV, bool SPLIT, bool ONCE>
__global__ void __launch_bounds__(fwd_shape(BF16).waves * 64, SPLIT ? fwd_shape(BF16).eu : 1) fwd_kernel(const FwdArgs p, const Board board) {
    constexpr int NW = fwd_shape(BF16).waves, RW = fwd_shape(BF16).rows, CH = NW * RW, E = BF16 ? 2 : 4;
    typedef RowVec<BF16, V> Vec;
    __shared__ Pair<V> agg[NW][64];
    __shared__ int cut[NW];
    __shared__ float last[64 * V];
    __shared__ int ticket;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = SPLIT ? blockIdx.x % board.slices : blockIdx.x;
    const int c0 = (slice * 64 + lane) * V;
    const bool active = c0 < p.C;
    const int c = c0 < p.C - V ? c0 : p.C - V;        // (with an odd C the last two lanes in it share a channel, with the same values)
    const int nchunks = (p.T + CH - 1) / CH;
    const int k = SPLIT ? take_ticket(board, slice, &ticket) : 0;
    float K[V];
#pragma unroll
    for (int v = 0; v < V; ++v) K[v] = SPLIT ? board.K[c + v] : p.scale * softplus_f32(param_at(p.decay, c + v, p.w_bf16));
    const bool near = all_near<V>(K);
    pass_empty(p.cu, p.S, p.C, p.initial, p.state, k * NW + wave, SPLIT ? nchunks * NW : NW, c, V, active);
    if (k >= nchunks) return;
    const int q0 = k * CH + wave * RW;
    Rows<REV, RW> rows;
    rows.set(q0, p.T);
    Vec xv[RW], rv[RW], iv[RW];
    {
        const rsrc_t xr = rows.at(p.x, p.xs), gr = rows.at(p.gates, p.gs);
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            rv[r].template bload<ONCE ? 2 : 0>(gr, c * E, rows.off(r, (int)p.gs));
            iv[r].template bload<ONCE ? 2 : 0>(gr, c * E, rows.off(r, (int)p.gs) + p.C * E);
            xv[r].template bload<ONCE ? 2 : 0>(xr, c * E, rows.off(r, (int)p.xs));
        }
    }
    Edges<REV, RW> ed;
    ed.locate(p.cu, p.S, q0, p.T);
    const uint32_t starts = ed.bits & ((1u << RW) - 1);
    const int n = rows.n;
    const bool plain = n == RW && !starts;
    // the state as if nothing came before the wave (or before the last start), and the product of the decays since then
    float h[RW][V], P[RW][V];
    auto scan = [&](auto all, auto near) {
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float x[V], rg[V], ig[V];
            stay<all.value + near.value>(xv[r]), stay<all.value + near.value>(rv[r]), stay<all.value + near.value>(iv[r]);
            xv[r].to_f32(x);
            rv[r].to_f32(rg);
            iv[r].to_f32(ig);
            const bool real = all || r < n, on = r && (all || !(starts >> r & 1));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float sr, z, u, a;
                decay_of<near.value>(rg[v], K[v], sr, z, u, a);
                const float beta = __builtin_amdgcn_sqrtf(fmaf(-u, u, u + u));
                float b = beta * sigmoid_f32(ig[v]) * x[v];
                if (!real) a = 1.f, b = 0.f;
                h[r][v] = on ? fmaf(a, h[r ? r - 1 : 0][v], b) : b;
                P[r][v] = on ? a * P[r ? r - 1 : 0][v] : a;
            }
        }
    };
    if (plain && near) scan(std::true_type{}, std::true_type{});
    else if (plain) scan(std::true_type{}, std::false_type{});
    else scan(std::false_type{}, std::false_type{});
    Pair<V> mine;
#pragma unroll
    for (int v = 0; v < V; ++v) mine.A[v] = left_of(P[RW - 1][v]), mine.B[v] = h[RW - 1][v];
    if (starts && p.initial) {
        float h0[V];
        load_f32<V>(h0, p.initial, ed.entered(31 - __builtin_clz(starts)), p.S, p.C, c);
#pragma unroll
        for (int v = 0; v < V; ++v) mine.B[v] = fmaf(mine.A[v], h0[v], mine.B[v]);
    }
    agg[wave][lane] = mine;
    if (lane == 0) cut[wave] = starts != 0;
    __syncthreads();
    if constexpr (SPLIT) {
        if (wave == 0) {
            Pair<V> all = mine;
            bool any = starts != 0;
            for (int w = 1; w < NW; ++w) {
                const Pair<V> f = agg[w][lane];
                const bool whole = cut[w] == 0;
                any |= !whole;
#pragma unroll
                for (int v = 0; v < V; ++v) all.A[v] = left_of(all.A[v] * f.A[v]), all.B[v] = whole ? fmaf(f.A[v], all.B[v], f.B[v]) : f.B[v];
            }
            int ks = k;                           // the chunk that the sequence of the first row began in
            if (!(starts & 1)) {
                const int qs = ed.before(0);
                ks = (qs < q0 ? qs : q0 - 1) / CH;
            }
            float front[V];
            look_back<V>(board, k, ks, all, any, c0, front);
#pragma unroll
            for (int v = 0; v < V; ++v) last[lane * V + v] = front[v];
        }
        __syncthreads();
    }
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = SPLIT ? last[lane * V + v] : 0.f;
    for (int w = 0; w < wave; ++w) {
        const Pair<V> f = agg[w][lane];
        const bool whole = cut[w] == 0;
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = whole ? fmaf(f.A[v], carry[v], f.B[v]) : f.B[v];
    }
    if (p.carries && active && wave * RW % kCarryRows == 0 && n > 0)
#pragma unroll
        for (int v = 0; v < V; ++v) p.carries[(size_t)(q0 / kCarryRows) * p.C + c + v] = carry[v];
    const rsrc_t yr = rows.at(p.y, (long long)p.C * E);
    if (plain) {
        bool endless = false;
#pragma unroll
        for (int v = 0; v < V; ++v) endless |= __builtin_isinf(carry[v]);
        if (__ballot(endless))
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) P[r][v] = left_of(P[r][v]);
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            Vec o;
#pragma unroll
            for (int v = 0; v < V; ++v) h[r][v] = fmaf(P[r][v], carry[v], h[r][v]);
            o.from_f32(h[r]);
            if (active) o.bstore(yr, c * E, rows.off(r, p.C * E));
        }
    } else {
        float from[V];
#pragma unroll
        for (int v = 0; v < V; ++v) from[v] = carry[v];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            if (starts >> r & 1) load_f32<V>(from, p.initial, ed.entered(r), p.S, p.C, c);
#pragma unroll
            for (int v = 0; v < V; ++v) h[r][v] = fmaf(left_of(P[r][v]), from[v], h[r][v]);
            Vec o;
            o.from_f32(h[r]);
            if (active && r < n) o.bstore(yr, c * E, rows.off(r, p.C * E));
        }
    }
    if (p.state && ed.bits >> 1 && n > 0) {
#pragma unroll
        for (int r = 0; r < RW; ++r)
            if (ed.bits >> (r + 1) & 1) {
                const int done = ed.left(r + 1);
                if (active) store_f32<V>(p.state, done, p.S, p.C, c, h[r]);
            }
    }
}

// The backward, chunks from the scan's end to its beginning. gamma is what comes back to a row's h from behind it:
// g_t = dy_t + gamma_t, gamma_{t-1} = a_t g_t. Every gradient is linear in g:
//   dx = g p1, di = g p2, m = g U (z times the gradient of z), dr = m (1 - sigmoid(r)),
// so that two passes over a wave's rows do: one that leaves p1, p2, U without the carry's part, sigmoid(r) and the decays of the rows and what the rows
// do to carry and gamma, and, when these are known, one that runs g and writes. p1 and p2 wait in the LDS in between: formed again from x and i instead they
// keep 32 more registers busy, and a third wave a SIMD spills. The forward's calls take 500 us (3.8 TB/s) and 153 us (4.6); the vector ALU is busy for half of it.
template <bool BF16, int V, bool REV, bool SPLIT, bool ONCE>
__global__ void __launch_bounds__(bwd_shape(BF16).waves * 64, SPLIT ? bwd_shape(BF16).eu : 1) bwd_kernel(const BwdArgs p, const Board board) {
    constexpr int NW = bwd_shape(BF16).waves, RW = bwd_shape(BF16).rows, CH = NW * RW, E = BF16 ? 2 : 4;
    static_assert(CH % kCarryRows == 0, "h is restarted once a chunk");
    typedef RowVec<BF16, V> Vec;
    typedef float Vals __attribute__((ext_vector_type(V == 1 ? 2 : V)));
    __shared__ Pair<V> fwd[NW - 1][64], bwd[NW][64];
    __shared__ Vals later[2][NW][RW][64];
    __shared__ int cut[NW];
    __shared__ float first[64 * V];
    __shared__ int ticket;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = SPLIT ? blockIdx.x % board.slices : blockIdx.x;
    const int c0 = (slice * 64 + lane) * V;
    const bool active = c0 < p.C;
    const int c = c0 < p.C - V ? c0 : p.C - V;        // (with an odd C the last two lanes in it share a channel, with the same values)
    const int nchunks = (p.T + CH - 1) / CH;
    const int k = SPLIT ? nchunks - 1 - take_ticket(board, slice, &ticket) : 0;
    float K[V];
#pragma unroll
    for (int v = 0; v < V; ++v) K[v] = SPLIT ? board.K[c + v] : p.scale * softplus_f32(param_at(p.decay, c + v, p.w_bf16));
    const bool near = all_near<V>(K);
    pass_empty(p.cu, p.S, p.C, p.dstate, p.dinitial, k * NW + wave, SPLIT ? nchunks * NW : NW, c, V, active);
    // ddecay's part of a chunk, or all of it
    auto leave = [&](float (&s)[V]) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (SPLIT) {
                p.partial[(size_t)k * p.C + c + v] = s[v];
                continue;
            }
            const float o = s[v] * softplus_ratio(param_at(p.decay, c + v, p.w_bf16));
            if (p.g_bf16) ((uint16_t*)p.ddecay)[c + v] = f32_to_bf16(o);
            else ((float*)p.ddecay)[c + v] = o;
        }
    };
    if (k >= nchunks) {
        float zero[V] = {};
        if (active && wave == 1) leave(zero);
        return;
    }
    const int q0 = k * CH + wave * RW;
    Rows<REV, RW> rows;
    rows.set(q0, p.T);
    Vec xv[RW], rv[RW], iv[RW], dv[RW];
    {
        const rsrc_t xr = rows.at(p.x, p.xs), gr = rows.at(p.gates, p.gs), dr = rows.at(p.dy, p.ds);
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            rv[r].template bload<ONCE ? 2 : 0>(gr, c * E, rows.off(r, (int)p.gs));
            iv[r].template bload<ONCE ? 2 : 0>(gr, c * E, rows.off(r, (int)p.gs) + p.C * E);
            xv[r].template bload<ONCE ? 2 : 0>(xr, c * E, rows.off(r, (int)p.xs));
        }
#pragma unroll
        for (int r = 0; r < RW; ++r) dv[r].template bload<ONCE ? 2 : 0>(dr, c * E, rows.off(r, (int)p.ds));
    }
    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = p.carries[(size_t)(k * (CH / kCarryRows)) * p.C + c + v];
    Edges<REV, RW> ed;
    ed.locate(p.cu, p.S, q0, p.T);
    const uint32_t starts = ed.bits & ((1u << RW) - 1);
    const int fs = starts ? __builtin_ctz(starts) : RW;           // rows in front of it continue what came before the wave
    const int n = rows.n;
    const bool plain = n == RW && !starts;
    const bool into = !(ed.bits >> RW & 1) && n == RW;            // something of the wave's last sequence comes behind it

    float sr[RW][V], U[RW][V], a[RW][V];
    Pair<V> f, b;
    // g of row r from g of the row behind it
    auto back = [&](auto way, int r, const float (&behind)[V], float (&g)[V]) {
        constexpr int L = RW - 1;
        float d[V];
        constexpr bool all = way.value > 0;
        stay<way.value>(dv[r]);
        dv[r].to_f32(d);
        const bool ends = ed.bits >> (r + 1) & 1;
        if (!all && r >= n)
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] = 0.f;
        if ((!all || r == L) && ends && p.dstate && r < n) {
            float e[V];
            load_f32<V>(e, p.dstate, ed.left(r + 1), p.S, p.C, c);
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] += e[v];
        }
        const bool on = r < L && (all || !ends);
#pragma unroll
        for (int v = 0; v < V; ++v) g[v] = on ? fmaf(a[r < L ? r + 1 : r][v], behind[v], d[v]) : d[v];
    };
    auto scan = [&](auto all, auto near) {
        float h[V], P[V];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
            float x[V], rg[V], ig[V], h0[V];
            Vals p1, p2;
            stay<all.value + near.value>(xv[r]), stay<all.value + near.value>(rv[r]), stay<all.value + near.value>(iv[r]);
            xv[r].to_f32(x);
            rv[r].to_f32(rg);
            iv[r].to_f32(ig);
            const bool real = all || r < n, start = !all && (starts >> r & 1);
            if (start) load_f32<V>(h0, p.initial, ed.entered(r), p.S, p.C, c);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float z, u, now;
                decay_of<near.value>(rg[v], K[v], sr[r][v], z, u, now);
                const float beta2 = fmaf(-u, u, u + u);
                const float ib = __builtin_amdgcn_rsqf(fmaxf(beta2, 1e-37f)), si = sigmoid_f32(ig[v]);
                a[r][v] = real ? now : 1.f;
                p1[v] = beta2 * ib * si;
                const float bt = real ? p1[v] * x[v] : 0.f;
                p2[v] = bt * (1.f - si);
                const float ai = a[r][v] * ib, za = z * a[r][v], zb = z * (bt * ai * ai);   // (z * bt may underflow)
                const float before = start ? h0[v] : r ? h[v] : 0.f, scaled = r && !start ? P[v] : 1.f;
                U[r][v] = real ? fmaf(-za, before, zb) : 0.f;
                h[v] = fmaf(a[r][v], before, bt);
                P[v] = a[r][v] * scaled;
            }
            later[0][wave][r][lane] = p1;
            later[1][wave][r][lane] = p2;
            // (what is left of the row, now: put off, its parts take more registers than it)
#pragma unroll
            for (int v = 0; v < V; ++v) asm volatile("" : "+v"(sr[r][v]), "+v"(U[r][v]), "+v"(a[r][v]));
        }
        float g[V], Q[V];
#pragma unroll
        for (int r = RW - 1; r >= 0; --r) {
            back(std::integral_constant<int, all.value + near.value>{}, r, g, g);
#pragma unroll
            for (int v = 0; v < V; ++v) Q[v] = r < RW - 1 ? a[r][v] * Q[v] : a[r][v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            f.A[v] = left_of(P[v]);
            f.B[v] = h[v];
            b.A[v] = starts & 1 ? 0.f : left_of(Q[v]);
            b.B[v] = starts & 1 ? 0.f : a[0][v] * g[v];
        }
    };
    if (plain && near) scan(std::true_type{}, std::true_type{});
    else if (plain) scan(std::true_type{}, std::false_type{});
    else scan(std::false_type{}, std::false_type{});
    if (wave < NW - 1) fwd[wave][lane] = f;
    bwd[wave][lane] = b;
    if (lane == 0) cut[wave] = starts != 0;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        const Pair<V> f = fwd[w][lane];
        const bool whole = cut[w] == 0;
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = whole ? fmaf(f.A[v], carry[v], f.B[v]) : f.B[v];
    }
    // what the carry adds to h_{t-1}: itself times the decays so far, until a sequence begins
#pragma unroll
    for (int r = 0; r < RW; ++r)
        if (r < fs && r < n)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                U[r][v] = fmaf(-(sr[r][v] * K[v] * a[r][v]), carry[v], U[r][v]);
                carry[v] *= a[r][v];
            }
    if constexpr (SPLIT) {
        if (wave == NW - 1) {
            Pair<V> all = b;
            bool any = starts != 0;
            for (int w = NW - 2; w >= 0; --w) {
                const Pair<V> f = bwd[w][lane];
                const bool whole = cut[w] == 0;
                any |= !whole;
#pragma unroll
                for (int v = 0; v < V; ++v) all.A[v] = left_of(all.A[v] * f.A[v]), all.B[v] = whole ? fmaf(f.A[v], all.B[v], f.B[v]) : f.B[v];
            }
            int ke = k;                           // the chunk that the sequence of the last row ends in
            if (into) {
                const int qe = ed.behind(RW);
                ke = (qe > q0 + RW ? qe - 1 : q0 + RW) / CH;
            }
            float behind[V];
            look_back<V>(board, nchunks - 1 - k, nchunks - 1 - ke, all, any, c0, behind);
#pragma unroll
            for (int v = 0; v < V; ++v) first[lane * V + v] = behind[v];
        }
        __syncthreads();
    }
    float gamma[V];
#pragma unroll
    for (int v = 0; v < V; ++v) gamma[v] = SPLIT ? first[lane * V + v] : 0.f;
    for (int w = NW - 1; w > wave; --w) {
        const Pair<V> f = bwd[w][lane];
        const bool whole = cut[w] == 0;
#pragma unroll
        for (int v = 0; v < V; ++v) gamma[v] = whole ? fmaf(f.A[v], gamma[v], f.B[v]) : f.B[v];
    }
    if (!into)                                    // (and keep a non-finite one of another sequence away)
#pragma unroll
        for (int v = 0; v < V; ++v) gamma[v] = 0.f;
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.f;
    const rsrc_t xr = rows.at(p.dx, (long long)p.C * E), gr = rows.at(p.dgates, 2ll * p.C * E);
    auto finish = [&](auto all) {                 // (a way of its own: the rows of dy are not to be kept widened since the scan)
        float g[V];
#pragma unroll
        for (int r = RW - 1; r >= 0; --r) {
            float dx[V], dr[V], di[V];
            back(all, r, g, g);
            const Vals p1 = later[0][wave][r][lane], p2 = later[1][wave][r][lane];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (r == RW - 1) g[v] += gamma[v];
                const float m = g[v] * U[r][v];
                sum[v] += m;
                dx[v] = g[v] * p1[v];
                dr[v] = m * (1.f - sr[r][v]);
                di[v] = g[v] * p2[v];
            }
            if (active && (all || r < n)) {
                Vec o;
                o.from_f32(dx);
                o.bstore(xr, c * E, rows.off(r, p.C * E));
                o.from_f32(dr);
                o.bstore(gr, c * E, rows.off(r, 2 * p.C * E));
                o.from_f32(di);
                o.bstore(gr, c * E, rows.off(r, 2 * p.C * E) + p.C * E);
            }
            if (!all && p.dinitial && (starts >> r & 1) && r < n) {
                const int begun = ed.entered(r);
                float d[V];
#pragma unroll
                for (int v = 0; v < V; ++v) d[v] = a[r][v] * g[v];
                if (active) store_f32<V>(p.dinitial, begun, p.S, p.C, c, d);
            }
        }
    };
    if (plain) finish(std::integral_constant<int, 3>{}); else finish(std::integral_constant<int, 0>{});
    // (the waves' carries are read in front of the last barrier, their sums written behind it)
    if (!SPLIT) __syncthreads();
    static_assert(2 * (NW - 1) >= NW, "the sums fit");
    float* const sums = (float*)fwd;
#pragma unroll
    for (int v = 0; v < V; ++v) sums[(wave * 64 + lane) * V + v] = sum[v];
    __syncthreads();
    if (wave == 1 && active) {
        float s[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v] = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) s[v] += sums[(w * 64 + lane) * V + v];
        }
        leave(s);
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

// One token of each of B sequences. A block has a row and 256 channels of it. The row that names a slot first also computes the later
// rows that name it, in their order; they do nothing. To find them out, a block reads all B slots (at C=2048 a quarter of the time of 512 rows, 10 us, three
// quarters of that of 8192, 0.3 ms), and where there are any it goes from one to the next a slot at a time (512 rows, four a slot: 69 us).
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
        float x[1], r[1], i[1], sr, z, u, a;
        xv.to_f32(x);
        rv.to_f32(r);
        iv.to_f32(i);
        decay_of<false>(r[0], K, sr, z, u, a);
        h = fmaf(a, h, __builtin_amdgcn_sqrtf(fmaf(-u, u, u + u)) * sigmoid_f32(i[0]) * x[0]);
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
