// Kernels of linear attention with a decay for each head (include/nplm_linattn.h).
//
// With b_i the sum of the log decays of rows up to i (counted from wherever a chunk begins) and S the state in front of a chunk (64 rows, 32 of fp32),
//
//   o_i  = scale * ( sum_{j <= i} e^(b_i - b_j) (q_i . k_j) v_j  +  e^(b_i) q_i S )
//   S'   = e^(b_end) S + sum_j e^(b_end - b_j) k_j v_j^T
//
// so a chunk is six matrix products, and rows are read once and written once. A block has one head of one segment, up to L rows of one sequence, and
// goes through its chunks with the state in registers. Where a sequence has more than one segment, the states at the boundaries come first: what each
// segment adds on its own (local_kernel), then one pass along the boundaries (scan_kernel).
//
// The gradients are the same products. With dS the gradient of the state behind a chunk,
//
//   dq_i = scale * ( sum_{j <= i} e^(b_i - b_j) (do_i . v_j) k_j  +  e^(b_i) do_i S^T )                    walk_kernel with (do, v, k) in place of (q, k, v)
//   dv_j = sum_{i >= j} e^(b_i - b_j) scale (q_i . k_j) do_i  +  e^(b_end - b_j) k_j dS                    back_kernel, chunks from the last to the first
//   dk_j = sum_{i >= j} e^(b_i - b_j) scale (do_i . v_j) q_i  +  e^(b_end - b_j) v_j dS^T
//   dS'  = e^(b_end) dS + sum_i e^(b_i) scale q_i do_i^T
//
// and log a_t collects every product that crosses row t: with e_i = (products that i reads from rows before it) - (products of i that rows behind it read),
// d/dlog a_t = sum_{i >= t} e_i + <S, dS> at the segment's end. A row's product with itself is in neither, so nothing is left of it to cancel.
//
// Matrix instructions are 16 x 16 (v_mfma_f32_16x16x32_bf16, or four v_mfma_f32_16x16x4_f32): lane l holds row or column l % 16 of an operand at
// the contraction's places of group l / 16, and column l % 16, rows 4 (l / 16) + 0 .. 3 of a result. A result's lane thus has four adjacent places of a
// contraction over its rows: the state goes back in as an operand without leaving its registers, if the other operand is read at the same places.
#pragma once
#include "dwconv_device.h"

namespace nplm {
namespace la {

// Rows of a chunk. fp32 has half as many: the backward's four tiles of 128 channels and two of scores would not fit LDS.
constexpr int chunk_rows(bool bf16) { return bf16 ? 64 : 32; }

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

struct Tensor3 {                     // [T, H, d], adjacent elements; strides in bytes
    const char* p;
    long long row, head;
    int vec;                         // whether every 16 bytes of it can be one load
};
struct States {                      // [n, H, keys, values] of some tensor, or its transpose
    int sk, sv;                      // elements from one contraction place (key side) to the next, from one column to the next
};
struct Shape {
    const int32_t* cu;
    const char* g;                   // log decays
    long long g_row, g_head;         // bytes; row 0 where a head has one
    int g_bf16, T, H, S, L, reverse;
};
struct WalkArgs {
    Shape s;
    Tensor3 q, k, v, x;              // x: what u multiplies
    char* out;
    const float *initial, *bound;
    float *last, *u;                 // u: [H, T]
    States st;
    float scale;
    int dk, dv;
};
struct BackArgs {
    Shape s;
    Tensor3 q, k, v, o;              // o: the gradient of the output
    char *dk_out, *dv_out;
    const float *dstate, *gbound, *state, *bound, *initial, *u;
    float *dinitial;
    char* dg;                        // [T, H], or
    double* dg_part;                 // [slots, H]
    int dg_bf16;
    float scale;
    int dk, dv;
};
struct LocalArgs {
    Shape s;
    Tensor3 k, v;
    float *bound, *decay;            // [T / L + 1, H, ...], [T / L + 1, H]
    States st;
    float scale;
    int dk, dv, back;
};
struct ScanArgs {
    Shape s;
    const float *edge;               // initial states or the last states' gradient, or null
    float *bound;
    const float *decay;
    int n, back, by_sequence;        // n: elements of a state
};
struct StepArgs {
    Tensor3 q, k, v;
    const char* g;
    long long g_row, g_head;
    int g_bf16;
    const float* state;
    float* out_state;
    const int32_t* slots;
    char* o;
    float scale;
    int B, H, dk, dv, bf16;
    long long N;
};

// ---- which rows a block has -----------------------------------------------------------------------------------------------------------
// The rows in front of cu[0] and behind cu[S] count as one sequence more on either side: sequence e of S + 2 is rows [edge(e), edge(e + 1)). It owns the
// places edge(e) / L + e and following of a launch, one for each segment of L rows: a sequence's segments never reach the next one's first place, and a block finds its
// sequence without a table. Everything is held within [0, T], whatever cu says.
__host__ __device__ __forceinline__ int edge_of(const Shape& s, long long e) {
    if (e <= 0) return 0;
    if (e > s.S + 1) return s.T;
    const int v = s.cu[e - 1];
    return v < 0 ? 0 : v > s.T ? s.T : v;
}
// The last e in [0, S + 1] with edge(e) / L + e <= place (segments) or edge(e) <= place (rows); the wave tries 64 of them at a time.
__host__ __device__ __forceinline__ int find_sequence(const Shape& s, long long place, bool segments) {
    long long lo = 0, n = (long long)s.S + 2;                  // the answer lies in [lo, lo + n)
#if defined(__HIP_DEVICE_COMPILE__)
    const int lane = threadIdx.x & 63;
#endif
    while (n > 1) {
        const long long step = (n + 63) >> 6;
        auto in = [&](int probe) {
            const long long e = lo + probe * step;
            return probe * step < n && (segments ? (long long)(edge_of(s, e) / s.L) + e : (long long)edge_of(s, e)) <= place;
        };
#if defined(__HIP_DEVICE_COMPILE__)
        const uint64_t m = __ballot(in(lane));
#else
        uint64_t m = 0;
        for (int probe = 0; probe < 64; ++probe) m |= (uint64_t)in(probe) << probe;
#endif
        const int f = 63 - __builtin_clzll(m | 1);             // (the first probe holds: edge(0) = 0)
        lo += f * step;
        n = n - f * step < step ? n - f * step : step;
    }
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_readfirstlane((int)lo);
#else
    return (int)lo;
#endif
}
struct Segment {
    int seq, lo, hi, p0, n;          // sequence (its number in cu; -1 and S: none), its rows, the segment's first place in it, its rows
    __host__ __device__ __forceinline__ long long row(const Shape& s, int p) const { return s.reverse ? hi - 1 - (p0 + p) : lo + p0 + p; }
    __host__ __device__ __forceinline__ bool last() const { return p0 + n >= hi - lo; }
    __host__ __device__ __forceinline__ long long bound(const Shape& s) const { return (lo + (long long)p0) / s.L; }             // of its first row, if that is not the sequence's
    __host__ __device__ __forceinline__ bool real(const Shape& s) const { return seq >= 0 && seq < s.S; }
};
__host__ __device__ __forceinline__ Segment segment_at(const Shape& s, long long place) {
    const int e = find_sequence(s, place, true);
    Segment g;
    g.seq = e - 1;
    g.lo = edge_of(s, e);
    g.hi = edge_of(s, (long long)e + 1);
    const long long p0 = (place - (g.lo / s.L + (long long)e)) * s.L;
    const int len = g.hi > g.lo ? g.hi - g.lo : 0;
    g.n = p0 < 0 || p0 >= len ? 0 : len - p0 < s.L ? (int)(len - p0) : s.L;
    g.p0 = p0 < 0 || p0 > len ? len : (int)p0;
    if (len == 0 && p0 != 0) g.seq = -1;                       // (an empty sequence's state is its first place's)
    return g;
}
// Boundary i in [1, T / L]: there is at most one first row r of a later segment with r / L = i, and it is of the sequence that has row i L - 1.
// The segment behind it; n is 0 where there is none.
__host__ __device__ __forceinline__ Segment boundary(const Shape& s, long long i) {
    const long long at = i * s.L - 1;
    const int e = find_sequence(s, at, false);
    Segment g;
    g.seq = e - 1;
    g.lo = edge_of(s, e);
    g.hi = edge_of(s, (long long)e + 1);
    const long long p0 = (at + s.L - g.lo) / s.L * s.L, len = (long long)g.hi - g.lo;
    const bool there = g.lo <= at && p0 < len;
    g.p0 = there ? (int)p0 : 0;
    g.n = !there ? 0 : len - p0 < s.L ? (int)(len - p0) : s.L;
    return g;
}

// ---- operands of the matrix instructions ----------------------------------------------------------------------------------------------
// The lane's number, each time as if it were new: addresses that are made of it are made again where they are used (a few instructions) and not once for the whole
// loop, whose registers they would fill.
__device__ __forceinline__ int this_lane() {
    int l = threadIdx.x & 63;
    asm volatile("" : "+v"(l));
    return l;
}
typedef uint32_t u32_pair __attribute__((ext_vector_type(2)));
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float lane_sum4(float v) {         // over lanes xor 16, 32
    u32_pair r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r.x) + __uint_as_float(r.y);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}
__device__ __forceinline__ float lane_sum16(float v) {        // over the 16 lanes of a group
    v += dpp<0xB1>(v);                                        // lanes xor 1, xor 2, the other half of 8, the other half of 16
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}
template <bool BF16> struct Op;
template <> struct Op<true> {
    static constexpr int KS = 32, E = 2, CH = chunk_rows(true), SCORES = 12;
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    // The 16 x 16 tiles of scores that are looked at (reading rows it, rows read jt): those on and below the diagonal, and above it what fills a contraction of 32
    // with zeros. by_reader: whether the contraction runs over the rows read (forward) or over the readers.
    static __device__ __forceinline__ void score(int t, bool by_reader, int& it, int& jt) {
        it = by_reader ? (t < 4 ? t >> 1 : 2 + ((t - 4) >> 2)) : t < 8 ? t & 3 : 2 + ((t - 8) & 1);
        jt = by_reader ? (t < 4 ? t & 1 : (t - 4) & 3) : t < 8 ? t >> 2 : 2 + ((t - 8) >> 1);
    }
    static __device__ __forceinline__ constexpr int reads_to(int it) { return it < 2 ? 32 : 64; }     // where the contraction of reading rows it ends,
    static __device__ __forceinline__ constexpr int read_from(int jt) { return jt < 2 ? 0 : 32; }     // where that of rows jt begins
    // 0, or NaN where an element is not finite
    static __device__ __forceinline__ float zero_of(frag v) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        const pair none = {(__bf16)0.f, (__bf16)0.f};
        float a = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(v, v, 0, 1), none, 0.f, false), b = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(v, v, 2, 3), none, 0.f, false);
        a = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(v, v, 4, 5), none, a, false);
        b = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(v, v, 6, 7), none, b, false);
        return a + b;
    }
};
template <> struct Op<false> {
    static constexpr int KS = 16, E = 4, CH = chunk_rows(false), SCORES = 3;
    typedef f32x4 frag;
    static __device__ __forceinline__ void score(int t, bool, int& it, int& jt) { it = t > 0, jt = t > 1; }
    static __device__ __forceinline__ constexpr int reads_to(int it) { return it * 16 + 16; }
    static __device__ __forceinline__ constexpr int read_from(int jt) { return jt * 16; }
    static __device__ __forceinline__ float zero_of(frag v) { return fmaf(v[1], 0.f, v[0] * 0.f) + fmaf(v[3], 0.f, v[2] * 0.f); }
    static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// A chunk's rows of D elements in LDS. Pieces of 16 bytes are exchanged within a row by its number, so that 16 rows of one column (operands by row, of 8 or 16
// bytes a lane) and 32 bytes each of rows 0 .. 3 and 8 .. 11 (or 4 .. 7 and 12 .. 15; operands by column) lie on all different banks.
template <bool BF16, int D> struct Tile {
    typedef Op<BF16> O;
    typedef typename O::frag frag;
    static constexpr int E = O::E, STRIDE = D * E, BYTES = O::CH * STRIDE;
    char* p;
    static __device__ __forceinline__ int swizzle(int row) {       // bytes
        if constexpr (STRIDE == 64) return (row >> 2 & 3) << 4;
        else if constexpr (STRIDE == 128) return ((row >> 2 & 1) | (row & 2) | (row >> 1 & 4)) << 4;
        else return ((row >> 2 & 1) | (row & 3) << 1 | (row & 8)) << 4;
    }
    __device__ __forceinline__ char* at(int row, int byte) const { return p + row * STRIDE + (byte ^ swizzle(row)); }
    // l: the lane. Its row row0 + l % 16, adjacent contraction places from k0 on: KS / 4 of group l / 16
    __device__ __forceinline__ frag rows(int l, int row0, int k0) const {
        return *(const frag*)at(row0 + (l & 15), (k0 + (l >> 4) * (O::KS / 4)) * E);
    }
    // the same at the places that a result has its rows: 4 of group l / 16 in each 16
    __device__ __forceinline__ frag rows_as_result(int l, int row0, int k0) const {
        const int row = row0 + (l & 15);
        if constexpr (BF16) {
            const bf16x4 a = *(const bf16x4*)at(row, (k0 + (l >> 4) * 4) * E), b = *(const bf16x4*)at(row, (k0 + 16 + (l >> 4) * 4) * E);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *(const frag*)at(row, (k0 + (l >> 4) * 4) * E);
        }
    }
    // its column c0 + l % 16, contraction over rows from k0 on: KS / 4 adjacent ones of group l / 16
    __device__ __forceinline__ frag columns(int l, int k0, int c0) const {
        if constexpr (BF16) {                                  // (the instruction gives lane i of 16 column i of the 4 x 16 elements that the 16 lanes point at)
            const int row = k0 + (l >> 4) * 8 + ((l & 15) >> 2), byte = (c0 + (l & 3) * 4) * E;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at(row, byte)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at(row + 4, byte));
            return __builtin_bit_cast(frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int row = k0 + (l >> 4) * 4, byte = (c0 + (l & 15)) * E;
            return (frag){*(const float*)at(row, byte), *(const float*)at(row + 1, byte), *(const float*)at(row + 2, byte), *(const float*)at(row + 3, byte)};
        }
    }
    // an element
    __device__ __forceinline__ float element(int row, int c) const {
        const char* const e = at(row, c * E);
        if constexpr (BF16) return bf16_to_f32(*(const uint16_t*)e);
        else return *(const float*)e;
    }
    // four adjacent columns of a row
    __device__ __forceinline__ f32x4 quad(int row, int c) const { return quad_at(at(row, c * E)); }
    __device__ __forceinline__ void put_quad(int row, int c, f32x4 v) const { put(at(row, c * E), v); }
    static __device__ __forceinline__ f32x4 quad_at(const char* at) {
        if constexpr (BF16) {
            const u32x2 u = *(const u32x2*)at;
            return (f32x4){bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)};
        } else {
            return *(const f32x4*)at;
        }
    }
    static __device__ __forceinline__ void put(char* at, f32x4 v) {
        if constexpr (BF16) *(u32x2*)at = (u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else *(f32x4*)at = v;
    }
};

// An fp32 operand as the instruction takes it: itself, or its bf16 rounding, the rounding of what that leaves, and so on: TERMS of them keep 8, 16 or 24 bits.
// One term rounds as the scores are rounded (half a step of bf16, 2^-9 of it) and is what rows that serve results in bf16 are added to the state with. The state
// that rows read has two: with one, o of 131072 rows of 16 heads of 64 was 2.5e-3 off (2-norm; the rounding of o alone is 1.7e-3), with two 2.3e-3, for 10 us of 257.
// Two are also for all that the gradients of bf16 log decays come from, sums over up to a segment's rows of terms that cancel: with one 5.4e-3 off, with two
// 1.7e-3, a rounding. Three are for results in fp32: states handed out, gradients of initial states and of fp32 log decays.
template <bool BF16, int TERMS> struct Split {
    typedef Op<BF16> O;
    static constexpr int N = BF16 ? 8 : 4, M = BF16 ? TERMS : 1;
    typename O::frag t[M];
    __device__ __forceinline__ void from(const float (&f)[N]) {
        if constexpr (BF16) {
            float left[N];
#pragma unroll
            for (int e = 0; e < N; ++e) left[e] = f[e];
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    t[m][e] = (__bf16)left[e];
                    if (m + 1 < M) left[e] -= (float)t[m][e];
                }
        } else {
            t[0] = (f32x4){f[0], f[1], f[2], f[3]};
        }
    }
    // a result's rows of 16 (32 in bf16) as contraction places
    __device__ __forceinline__ void from_result(const f32x4* r) {
        float f[N];
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = r[e >> 2][e & 3];
        from(f);
    }
    // an operand times a weight for each of its contraction places, rows k0 on
    __device__ __forceinline__ void weighted(int l, typename O::frag v, const float* w, int k0) {
        const int g = l >> 4;
        const f32x4* at = (const f32x4*)(w + k0 + g * N);
        float f[N];
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = (float)v[e] * at[e >> 2][e & 3];
        from(f);
    }
    template <bool FIRST> __device__ __forceinline__ f32x4 times(typename O::frag other, f32x4 c) const {      // FIRST: this one is the first operand
#pragma unroll
        for (int m = M - 1; m >= 0; --m) c = FIRST ? O::mma(t[m], other, c) : O::mma(other, t[m], c);
        return c;
    }
};

// ---- rows on their way into LDS -------------------------------------------------------------------------------------------------------
// A tensor's rows of a segment and head as a buffer: what lies outside of them reads as 0 and is not written, whatever the row's number, so rows need no
// tests. Offsets stay below 2^30 from end to end (the host sees to that: VEC); columns that do not exist point beyond all of it.
constexpr uint32_t kNowhere = 0x80000000u;
struct Rows {
    rsrc_t r;
    uint32_t first;                  // offset of the segment's first row
    int step;                        // from a row to the next one in the walk's order
    __device__ __forceinline__ Rows(const char* p, long long row, long long head, const Shape& s, const Segment& g, int h, int bytes) {
        const long long low = s.reverse ? (long long)g.hi - g.p0 - g.n : (long long)g.lo + g.p0;
        r = make_rsrc(p + low * row + h * head, g.n > 0 ? (uint32_t)((g.n - 1) * row + bytes) : 0u);
        first = s.reverse ? (uint32_t)((g.n - 1) * row) : 0u;
        step = s.reverse ? -(int)row : (int)row;
    }
    __device__ __forceinline__ uint32_t at(int row, int c, int bytes) const { return c < bytes ? first + (uint32_t)(row * step + c) : kNowhere; }
};
// NT threads' share of a chunk's rows of D elements (of which d exist), 16 bytes at a time, from chunk to chunk. What a thread puts into a tile (Fetch) and
// what it takes out of it to memory (Drain) are the same places.
template <bool BF16, int D, int NT> struct Share {
    static constexpr int E = BF16 ? 2 : 4, PER = 16 / E, UR = D * E / 16, CH = chunk_rows(BF16), N = CH * UR / NT, APART = NT / UR;
    static_assert(N * NT == CH * UR && NT % UR == 0, "whole units, a thread's all of the same columns");
    static __device__ __forceinline__ int unit_row(int i) { return (int)(threadIdx.x + i * NT) / UR; }
    static __device__ __forceinline__ int unit_byte() { return (int)threadIdx.x % UR * 16; }
    // as if it were new each time (this_lane): addresses of 64 bits
    static __device__ __forceinline__ int this_thread() {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        return t;
    }
};
// 16 bytes that lie at their element's alignment
template <bool BF16> struct Loose;
template <> struct Loose<true> { typedef u32x4 type __attribute__((aligned(2))); typedef uint16_t word; };
template <> struct Loose<false> { typedef u32x4 type __attribute__((aligned(4))); typedef uint32_t word; };

template <bool BF16, int D, int NT, bool VEC> struct Fetch : Share<BF16, D, NT> {
    typedef Share<BF16, D, NT> Sh;
    u32x4 r[Sh::N];
    Rows rows;
    uint32_t off;                    // of the first unit; the others lie NT / UR rows apart
    __device__ __forceinline__ Fetch(const Tensor3& t, const Shape& s, const Segment& g, int h, int d, int p0) : rows(t.p, t.row, t.head, s, g, h, d * Sh::E) {
        if constexpr (VEC) off = rows.at(p0 + Sh::unit_row(0), Sh::unit_byte(), d * Sh::E);
    }
    // the chunk from place p0 on; the next one is behind it (forward) or in front of it
    __device__ __forceinline__ void load(const Tensor3& t, const Shape& s, const Segment& g, int h, int p0, int d, bool forward) {
        if constexpr (VEC) {
            const uint32_t next = (uint32_t)(forward ? Sh::CH * rows.step : -Sh::CH * rows.step);
#pragma unroll
            for (int i = 0; i < Sh::N; ++i) r[i] = __builtin_amdgcn_raw_buffer_load_b128(rows.r, off + (uint32_t)(i * Sh::APART * rows.step), 0, 0);
            off += next;
            return;
        }
        const int c = Sh::unit_byte() / Sh::E;
        if (d < Sh::PER) {                                     // (uniform) rows shorter than 16 bytes
#pragma unroll 1
            for (int i = 0; i < Sh::N; ++i) {
                const int p = p0 + Sh::unit_row(i);
                u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll 1
                for (int e = 0; e < d; ++e)
                    if (c == 0 && p < g.n) {
                        const uint32_t x = ((const typename Loose<BF16>::word*)(t.p + g.row(s, p) * t.row + h * t.head))[e];
                        if constexpr (BF16) v[e >> 1] |= x << (e & 1) * 16; else v[e] = x;
                    }
#pragma unroll
                for (int j = 0; j < Sh::N; ++j) r[j] = i == j ? v : r[j];
            }
            return;
        }
        // a row's last unit reads back from its end, and moves down what it has on its way into LDS
        const int me = Sh::this_thread(), row = me / Sh::UR, unit = me % Sh::UR * Sh::PER, left = d - unit, back = left > 0 && left < Sh::PER ? Sh::PER - left : 0;
        const char* const at = t.p + g.row(s, p0 + row) * t.row + h * t.head + (unit - back) * Sh::E;
        const long long apart = s.reverse ? -Sh::APART * t.row : Sh::APART * t.row;
#pragma unroll
        for (int i = 0; i < Sh::N; ++i) {
            u32x4 v = {0u, 0u, 0u, 0u};
            if (p0 + row + i * Sh::APART < g.n && left > 0) v = *(const typename Loose<BF16>::type*)(at + i * apart);
            r[i] = v;
        }
    }
    __device__ __forceinline__ void store(const Tile<BF16, D>& t, int d) const {
        const int have = VEC ? 0 : d - Sh::this_thread() % Sh::UR * Sh::PER, back = d > Sh::PER && have > 0 && have < Sh::PER ? Sh::PER - have : 0, q = back * Sh::E >> 2;
#pragma unroll
        for (int i = 0; i < Sh::N; ++i) {
            u32x4 v = r[i];
            if (!VEC && d % Sh::PER) {
                v = (q & 1) ? (u32x4){v[1], v[2], v[3], 0u} : v;
                v = (q & 2) ? (u32x4){v[2], v[3], 0u, 0u} : v;
                if constexpr (BF16)
                    if (back & 1) v = (u32x4){v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
            }
            *(u32x4*)t.at(Sh::unit_row(i), Sh::unit_byte()) = v;
        }
    }
};
// A chunk's results from a tile to [T, H, d], 16 bytes a lane, so that a wave's stores fill whole lines. Straight from the registers a lane has 8 bytes and a wave 32 of a
// row, and the next chunk's loads waited behind such stores for most of the first kernels' time.
template <bool BF16, int D, int NT, bool VEC> struct Drain : Share<BF16, D, NT> {
    typedef Share<BF16, D, NT> Sh;
    u32x4 r[Sh::N];
    Rows rows;
    char* p;
    long long row;
    uint32_t off;                    // of the first unit; the others lie NT / UR rows apart
    __device__ __forceinline__ Drain(char* out, const Shape& s, const Segment& g, int h, int d, int p0)
        : rows(out, (long long)s.H * d * Sh::E, (long long)d * Sh::E, s, g, h, d * Sh::E), p(out + (long long)h * d * Sh::E), row((long long)s.H * d * Sh::E) {
        if constexpr (VEC) off = rows.at(p0 + Sh::unit_row(0), Sh::unit_byte(), d * Sh::E);
    }
    // out of the tile, and to memory: loads that a wave waits for in between are not waited for together with these stores
    __device__ __forceinline__ void take(const Tile<BF16, D>& t) {
#pragma unroll
        for (int i = 0; i < Sh::N; ++i) r[i] = *(const u32x4*)t.at(Sh::unit_row(i), Sh::unit_byte());
    }
    __device__ __forceinline__ void give(const Shape& s, const Segment& g, int p0, int d, bool forward) {
        const uint32_t next = (uint32_t)(forward ? Sh::CH * rows.step : -Sh::CH * rows.step);
        const int me = VEC ? 0 : Sh::this_thread(), c = me % Sh::UR * Sh::PER;
        const long long apart = s.reverse ? -Sh::APART * row : Sh::APART * row;
        char* const first = VEC ? nullptr : p + g.row(s, p0 + me / Sh::UR) * row + c * Sh::E;
#pragma unroll
        for (int i = 0; i < Sh::N; ++i) {
            if constexpr (VEC) {
                __builtin_amdgcn_raw_buffer_store_b128(r[i], rows.r, off + (uint32_t)(i * Sh::APART * rows.step), 0, kStoreAux);
            } else {
                if (p0 + me / Sh::UR + i * Sh::APART >= g.n || c >= d) continue;
                char* const to = first + i * apart;
                if (c + Sh::PER <= d) {
                    *(typename Loose<BF16>::type*)to = r[i];
                } else {
#pragma unroll
                    for (int e = 0; e + 1 < Sh::PER; ++e)
                        if (c + e < d) ((typename Loose<BF16>::word*)to)[e] = BF16 ? r[i][e >> 1] >> (e & 1) * 16 : r[i][e % 4];
                }
            }
        }
        if constexpr (VEC) off += next;
    }
};

// ---- decays of a chunk ----------------------------------------------------------------------------------------------------------------
// Log decays are summed in fp64, in units of log 2, and kept as two fp32 numbers: far into a chunk of strong decays the difference of two sums is
// what counts. One below -200 (e^-138, 0 in fp32) counts as -200, so that a state can be forgotten altogether and what follows is still exact.
// (read four at a time: the second of two as well)
template <int CH> struct alignas(16) Decays {
    float hi[CH], lo[CH];            // b
    float since[CH];                 // e^b, times scale
    float left[CH];                  // e^(b_end - b)
    float whole;                     // e^b_end
};
static_assert(sizeof(Decays<64>) % 16 == 0 && sizeof(Decays<32>) % 16 == 0, "pairs of them are aligned");
// A lane's row of a chunk in [T, H] (strides in bytes), from chunk to chunk.
struct RowPointer {
    const char* p;
    long long step;                  // from a chunk to the next one in the walk's order
    int place;
    __device__ __forceinline__ RowPointer(const void* base, long long row, long long head, const Shape& s, const Segment& g, int h, int place_, int chunk)
        : p((const char*)base + h * head + g.row(s, place_) * row), step(s.reverse ? -chunk * row : chunk * row), place(place_) {}
    __device__ __forceinline__ void next(int chunk) { p += step, place += chunk; }
    __device__ __forceinline__ void back(int chunk) { p -= step, place -= chunk; }
};
// A log decay as it lies in memory: what it is in fp32 is asked for when it is needed, behind the loads of the chunk that follow it.
__device__ __forceinline__ uint32_t raw_decay(const Shape& s, const RowPointer& r, int n, bool lane) {
    uint32_t v = 0;
    if (lane && r.place < n) {
        if (s.g_bf16) v = *(const uint16_t*)r.p;
        else v = *(const uint32_t*)r.p;
    }
    return v;
}
template <int CTRL, int ROWS> __device__ __forceinline__ double dpp_add(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false), hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xF, false);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);            // (lanes without a source add 0)
}
// Over the lanes of a wave, of which the first CH count: lanes 1, 2, 4, 8 before in 16, then the sums of the 16 and of the 32 before.
template <int CH> __device__ __forceinline__ double running_sum(double v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    if constexpr (CH == 64) v = dpp_add<0x143, 0xC>(v);
    return v;
}
// One wave, each lane its row's log decay (lanes beyond the chunk's rows 0); returns the sum over the chunk. scale goes into since.
template <int CH> __device__ __forceinline__ double chunk_decays(const Shape& s, uint32_t raw, Decays<CH>* d, float scale) {
    const int l = threadIdx.x & 63;
    double b = (double)__uint_as_float(s.g_bf16 ? raw << 16 : raw) * 1.4426950408889634;
    if (b < -200.0) b = -200.0;
    b = running_sum<CH>(b);
    const double end = __shfl(b, CH - 1);
    if (l < CH) {
        const float hi = (float)b;
        d->hi[l] = hi;
        d->lo[l] = (float)(b - (double)hi);
        d->since[l] = __builtin_amdgcn_exp2f(hi) * scale;
        d->left[l] = __builtin_amdgcn_exp2f((float)(end - b));
        if (l == 0) d->whole = __builtin_amdgcn_exp2f((float)end);
    }
    return end;
}

template <int N> struct Rows_ { static constexpr int value = N; };
// Whether a sequence's last chunk, if it has half of a chunk's rows or fewer, has half of the work: where registers are left for both ways. 131072 rows of 16 heads of 64 in
// sequences of 70, forward and backward 364 and 1225 us without, 332 and 1126 with it; 128 x 64 955 and 1139 (backward), fp32 152 and 176 (dq, 32768 rows of 12 heads).
constexpr bool halves(bool bf16, int dk, int dv) { return bf16 && dk <= 64 && dv <= 64; }

// What a wave does with a chunk: it has C x 16 columns of the result and of the state [R rows] for its own, reads rows of one tile against the state (queries; keys
// for dv, values for dk), weighs its columns of another (values; do for dv, queries for dk) by the scores, and adds these columns times rows of a third (keys; queries
// for dv, do for dk) to the state. An operand from LDS serves C instructions. FORWARD: from the first chunk to the last.
template <bool BF16, int R, int C, bool FORWARD> struct Role {
    typedef Op<BF16> O;
    typedef typename O::frag frag;
    static constexpr int CH = O::CH, KS = O::KS, SR = R / 16, PER = KS / 16, SF = SR / PER;
    // res[jt][c]: 16 rows of the result, transposed. own: the wave's columns of what the scores weigh. x (SUM): sums[j] is row j of x times what it read from the state
    // ROWS: how many of the chunk's there are at most, all or half.
    template <int TERMS, bool SUM, int ROWS, int N, int M, int D, int DX>
    static __device__ __forceinline__ void read(const f32x4 (&st)[N], f32x4 (&res)[M], frag (&of)[M], const Tile<BF16, R>& rows, const Tile<BF16, D>& own,
                                                const Tile<BF16, CH>& scores, const Tile<BF16, DX>& x, const Decays<CH>& d, int col0, float* sums, bool state) {
        const float* const weight = FORWARD ? d.since : d.left;
        const int l = this_lane(), lr = l & 15, lg = l >> 4;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < ROWS / KS; ++k) of[c * (CH / KS) + k] = own.columns(l, k * KS, col0 + c * 16);
#pragma unroll
        for (int i = 0; i < C * (CH / 16); ++i) res[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (state) {
#pragma unroll
            for (int t = 0; t < SF; ++t) {
                Split<BF16, TERMS> sf[C];
#pragma unroll
                for (int c = 0; c < C; ++c) sf[c].from_result(st + c * SR + t * PER);
#pragma unroll
                for (int jt = 0; jt < ROWS / 16; ++jt) {
                    const frag f = rows.rows_as_result(l, jt * 16, t * KS);
#pragma unroll
                    for (int c = 0; c < C; ++c) res[c * (CH / 16) + jt] = sf[c].template times<true>(f, res[c * (CH / 16) + jt]);
                }
            }
        }
        // Scores that are masked are zeros, and a zero times an infinity or NaN of a row that must not be read is NaN. The forward (and dq without the log decays' gradient) makes such
        // elements zeros to the instruction, too, and their products come one by one behind it. Looking for them in front of the products with the state, where a wave waits for
        // the rows, took 260 us in place of 255 (131072 rows of 16 heads of 64; 306 and 287 in sequences of 70), not at all 252 (284); 65536 rows of 16 heads of 128 280 and
        // 272. In the backward with wide keys it took 9 % (1098 to 1200 us) for gradients of what is not finite.
        float zero = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < ROWS / KS; ++k) zero += O::zero_of(of[c * (CH / KS) + k]);
        const bool broken = FORWARD && !SUM && __builtin_expect(__ballot(!(zero == 0.f)) != 0, 0);
        if (broken) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int k = 0; k < ROWS / KS; ++k)
#pragma unroll
                    for (int e = 0; e < (BF16 ? 8 : 4); ++e)
                        if (!__builtin_isfinite((float)of[c * (CH / KS) + k][e])) of[c * (CH / KS) + k][e] = 0;
        }
#pragma unroll
        for (int jt = 0; jt < ROWS / 16; ++jt) {
            const int j = jt * 16 + lr;
            const float left = weight[j];
            float w = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                f32x4& acc = res[c * (CH / 16) + jt];
                acc *= left;
                if constexpr (SUM) {
                    const f32x4 y = x.quad(j, col0 + c * 16 + lg * 4);
                    w += (acc[0] * y[0] + acc[1] * y[1]) + (acc[2] * y[2] + acc[3] * y[3]);
                }
            }
            if constexpr (SUM) {
                w = lane_sum4(w);
                if (lg == 0) sums[j] = w;
            }
#pragma unroll
            for (int k = FORWARD ? 0 : O::read_from(jt) / KS; k < (FORWARD ? O::reads_to(jt) : ROWS) / KS; ++k) {
                const frag f = scores.rows(l, jt * 16, k * KS);
#pragma unroll
                for (int c = 0; c < C; ++c) res[c * (CH / 16) + jt] = O::mma(of[c * (CH / KS) + k], f, res[c * (CH / 16) + jt]);
            }
        }
        if (broken) {
#pragma unroll 1
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const f32x4 y = own.quad(i, col0 + c * 16 + lg * 4);
#pragma unroll
                    for (int jt = 0; jt < ROWS / 16; ++jt) {
                        const int j = jt * 16 + lr;
                        const float p = scores.element(j, i);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if ((FORWARD ? i <= j : i >= j) && !__builtin_isfinite(y[r])) res[c * (CH / 16) + jt][r] += p * y[r];
                    }
                }
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int k = 0; k < ROWS / KS; ++k) of[c * (CH / KS) + k] = own.columns(l, k * KS, col0 + c * 16);
        }
    }
    template <int ROWS, int M, int D> static __device__ __forceinline__ void put(const f32x4 (&res)[M], const Tile<BF16, D>& to, int col0) {
        const int l = this_lane();
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int jt = 0; jt < ROWS / 16; ++jt) to.put_quad(jt * 16 + (l & 15), col0 + c * 16 + (l >> 4) * 4, res[c * (CH / 16) + jt]);
    }
    template <int TERMS, int ROWS, int N, int M>
    static __device__ __forceinline__ void add(f32x4 (&st)[N], const frag (&of)[M], const Tile<BF16, R>& columns, const Decays<CH>& d, const float* weight) {
        const int l = this_lane();
        const float whole = d.whole;
#pragma unroll
        for (int t = 0; t < SR * C; ++t) st[t] *= whole;
#pragma unroll
        for (int k = 0; k < ROWS / KS; ++k) {
            Split<BF16, TERMS> w[C];
#pragma unroll
            for (int c = 0; c < C; ++c) w[c].weighted(l, of[c * (CH / KS) + k], weight, k * KS);
#pragma unroll
            for (int t = 0; t < SR; ++t) {
                const frag f = columns.columns(l, k * KS, t * 16);
#pragma unroll
                for (int c = 0; c < C; ++c) st[c * SR + t] = w[c].template times<false>(f, st[c * SR + t]);
            }
        }
    }
    // the wave's part of a state, its rows sr and its columns sc elements apart
    template <int N> static __device__ __forceinline__ void load(f32x4 (&st)[N], const float* p, int sr, int sc, int nr, int nc, int col0) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int t = 0; t < SR; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = t * 16 + (l >> 4) * 4 + r, col = col0 + c * 16 + (l & 15);
                    st[c * SR + t][r] = row < nr && col < nc ? p[row * sr + col * sc] : 0.f;
                }
    }
    // <the wave's part of the state, another one in memory>, and the sum of the products' squares
    template <int N>
    static __device__ __forceinline__ void dot(const f32x4 (&st)[N], const float* p, int sr, int sc, int nr, int nc, int col0, double& sum, double& squares) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int t = 0; t < SR; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = t * 16 + (l >> 4) * 4 + r, col = col0 + c * 16 + (l & 15);
                    if (row < nr && col < nc) {
                        const double x = (double)st[c * SR + t][r] * (double)p[row * sr + col * sc];
                        sum += x, squares = fma(x, x, squares);
                    }
                }
    }
    template <int N> static __device__ __forceinline__ void save(const f32x4 (&st)[N], float* p, int sr, int sc, int nr, int nc, int col0) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int t = 0; t < SR; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = t * 16 + (l >> 4) * 4 + r, col = col0 + c * 16 + (l & 15);
                    if (row < nr && col < nc) p[row * sr + col * sc] = st[c * SR + t][r];
                }
    }
};

// Whether the differences of the sums of log decays take their second parts: for results in fp32. For results in bf16 what the first parts are off by goes under in the rounding of the
// score: with log decays of 0 or less a sum is -12800 at the least, either part of a difference is off by up to half a step there, 2^-11, a weight by up to 2^-10 ln 2 of it, below 2^-10.5,
// and usually below 2^-18.
template <bool BF16, int TERMS> constexpr bool fine() { return !BF16 || TERMS == 3; }

// ---- forward, and the gradient of the queries -----------------------------------------------------------------------------------------
// Bound by memory where there are blocks enough: 131072 rows of 16 heads of 64 in bf16, forward 250 us, 4.3 TB/s (as loads and stores alone 240 us), gradient 329 us (303).
// Heads of 128 are bound by instructions: vector ones 0.58 of the SIMDs' cycles and the products 0.32 (65536 rows of 16 heads in one sequence, states in three parts).
// Two columns of 16 a wave where keys and values are wide, an operand from LDS serves two products: 65536 rows of 16 heads of 128 with one 426 us, with two 357 (20011 rows of
// 8 heads of 64 and 128: 37 and 39).
// DG: with u_i = x_i . (what row i read from the state in front of its chunk).
template <bool BF16, int DK, int DV, int C, bool DG> struct WalkLds {
    char q[Tile<BF16, DK>::BYTES], k[Tile<BF16, DK>::BYTES], v[Tile<BF16, DV>::BYTES], p[Tile<BF16, chunk_rows(BF16)>::BYTES];
    char x[DG ? Tile<BF16, DV>::BYTES : 16];
    Decays<chunk_rows(BF16)> d[2];
    float u[DG ? DV / 16 / C : 1][chunk_rows(BF16)];
};
constexpr int walk_columns(int dk, int dv) { return dk == 128 && dv == 128 ? 2 : 1; }
template <bool BF16, int DK, int DV, int TERMS, bool DG, bool VEC>
__global__ void __launch_bounds__(DV * 4 / walk_columns(DK, DV), DK + DV == 128 && BF16 && !DG ? 4 : 2) walk_kernel(const WalkArgs a) {
    typedef Op<BF16> O;
    typedef typename O::frag frag;
    constexpr int C = walk_columns(DK, DV), NT = DV * 4 / C, NW = NT / 64, KS = O::KS, CH = O::CH;
    typedef Role<BF16, DK, C, true> W;
    __shared__ __attribute__((aligned(256))) WalkLds<BF16, DK, DV, C, DG> lds;
    const Tile<BF16, DK> tq{lds.q}, tk{lds.k};
    const Tile<BF16, DV> tv{lds.v}, tx{lds.x};
    const Tile<BF16, CH> tp{lds.p};
    const Shape& s = a.s;
    const int h = blockIdx.x % (unsigned)s.H, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
    const Segment g = segment_at(s, blockIdx.x / (unsigned)s.H);
    const int col0 = wave * 16 * C, n = a.dk * a.dv;
    const bool states = g.real(s);
    if (g.n == 0 && !(a.last && states && g.p0 == 0 && g.hi <= g.lo)) return;

    Fetch<BF16, DK, NT, VEC> fq(a.q, s, g, h, a.dk, 0), fk(a.k, s, g, h, a.dk, 0);
    Fetch<BF16, DV, NT, VEC> fv(a.v, s, g, h, a.dv, 0), fx(a.x, s, g, h, a.dv, 0);
    Drain<BF16, DV, NT, VEC> out(a.out, s, g, h, a.dv, 0);
    uint32_t decay = 0;
    RowPointer rate(s.g, s.g_row, s.g_head, s, g, h, l, CH);
    auto ask = [&](int p) {
        if (wave == 0) decay = raw_decay(s, rate, g.n, l < CH), rate.next(CH);
        fk.load(a.k, s, g, h, p, a.dk, true);
        fq.load(a.q, s, g, h, p, a.dk, true);
        fv.load(a.v, s, g, h, p, a.dv, true);
        if constexpr (DG) fx.load(a.x, s, g, h, p, a.dv, true);
    };
    if (g.n > 0) ask(0);
    f32x4 st[W::SR * C];
#pragma unroll
    for (int t = 0; t < W::SR * C; ++t) st[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const float* from = g.p0 > 0 ? a.bound : states ? a.initial : nullptr;
    const bool save = a.last && states && g.last();          // (nobody asks for the state behind the last chunk otherwise)
    if (from) W::load(st, from + ((g.p0 > 0 ? g.bound(s) : g.seq) * s.H + h) * (long long)n, a.st.sk, a.st.sv, a.dk, a.dv, col0);
    if (wave == 0) chunk_decays(s, decay, &lds.d[0], a.scale);
    for (int p = 0, now = 0; p < g.n; p += CH, now ^= 1) {
        const Decays<CH>& d = lds.d[now];
        __syncthreads();                                      // (everyone is through with the chunk before)
        if (p > 0) out.take(tv);
        fq.store(tq, a.dk), fk.store(tk, a.dk), fv.store(tv, a.dv);
        if constexpr (DG) fx.store(tx, a.dv);
        if (p > 0) out.give(s, g, p - CH, a.dv, true);
        __syncthreads();
        if (p + CH < g.n) ask(p + CH);
        const bool half = halves(BF16, DK, DV) && g.n - p <= CH / 2;
        // decayed scores, 16 x 16 at a time, those in front of or on the diagonal and those that fill a contraction of 32 with zeros
        for (int t = wave; t < O::SCORES; t += NW) {
            int it, jt;
            const int l = this_lane(), lr = l & 15, lg = l >> 4;
            O::score(t, true, it, jt);
            f32x4 c = {0.f, 0.f, 0.f, 0.f};
            const int i = it * 16 + lr, j = jt * 16 + lg * 4;
            if (it * 16 >= (half ? CH / 2 : CH)) continue;    // (nobody looks at it)
            if (jt > it) {
                tp.put_quad(i, j, c);
                continue;
            }
#pragma unroll
            for (int k = 0; k < DK; k += KS) c = O::mma(tk.rows(l, jt * 16, k), tq.rows(l, it * 16, k), c);
            f32x4 e = d.hi[i] - *(const f32x4*)(d.hi + j);
            if constexpr (fine<BF16, TERMS>()) e += d.lo[i] - *(const f32x4*)(d.lo + j);
#pragma unroll
            for (int r = 0; r < 4; ++r) c[r] *= __builtin_amdgcn_exp2f(e[r]) * a.scale;
            if (jt == it) {
                asm volatile("");                             // (a branch: three tiles of ten take it)
#pragma unroll
                for (int r = 0; r < 4; ++r) c[r] = j + r > i ? 0.f : c[r];
            }
            tp.put_quad(i, j, c);
        }
        __syncthreads();
        f32x4 res[C * (CH / 16)];
        frag of[C * (CH / 16)];
        auto read = [&](auto rows) {
            W::template read<DG ? TERMS : 2, DG, rows.value>(st, res, of, tq, tv, tp, tx, d, col0, DG ? lds.u[wave] : nullptr, p > 0 || from);
            W::template put<rows.value>(res, tv, col0);       // (over the wave's own columns of the values, which it has in of)
        };
        if (half) read(Rows_<CH / 2>{}); else read(Rows_<CH>{});
        if constexpr (DG) {
            __syncthreads();
            if (wave == NW - 1 && l < CH && p + l < g.n) {
                float u = 0.f;
#pragma unroll
                for (int w = 0; w < NW; ++w) u += lds.u[w][l];
                a.u[(long long)h * s.T + g.row(s, p + l)] = u;
            }
        }
        auto add = [&](auto rows) { W::template add<TERMS, rows.value>(st, of, tk, d, d.left); };
        if (p + CH < g.n || save) {
            if (half) add(Rows_<CH / 2>{}); else add(Rows_<CH>{});
        }
        if (wave == 0 && p + CH < g.n) chunk_decays(s, decay, &lds.d[now ^ 1], a.scale);
    }
    if (g.n > 0) {
        __syncthreads();
        out.take(tv);
        out.give(s, g, (g.n - 1) / CH * CH, a.dv, true);
    }
    if (save) W::save(st, a.last + ((long long)g.seq * s.H + h) * n, a.st.sk, a.st.sv, a.dk, a.dv, col0);
}

// ---- what a segment adds to the state on its own --------------------------------------------------------------------------------------
// Forward: of the segment in front of boundary i, sum_j e^(b_end - b_j) k_j v_j^T. back: of the segment behind it, sum_i e^(b_i) scale q_i do_i^T (k and v stand for q and do).
template <bool BF16, int DK, int DV, int TERMS, bool VEC>
__global__ void __launch_bounds__(DV * 4, 2) local_kernel(const LocalArgs a) {
    typedef Op<BF16> O;
    typedef typename O::frag frag;
    constexpr int C = 1, NT = DV * 4, KS = O::KS, CH = O::CH;
    typedef Role<BF16, DK, C, true> W;
    __shared__ __attribute__((aligned(256))) struct { char k[Tile<BF16, DK>::BYTES], v[Tile<BF16, DV>::BYTES]; Decays<CH> d[2]; } lds;
    const Tile<BF16, DK> tk{lds.k};
    const Tile<BF16, DV> tv{lds.v};
    const Shape& s = a.s;
    const int h = blockIdx.x % (unsigned)s.H, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, col0 = wave * 16 * C;
    const long long i = 1 + (long long)(blockIdx.x / (unsigned)s.H);
    Segment g = boundary(s, i);
    if (g.n == 0) return;
    if (!a.back) g.p0 -= s.L, g.n = s.L;
    f32x4 st[W::SR * C];
#pragma unroll
    for (int t = 0; t < W::SR * C; ++t) st[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int chunks = (g.n + CH - 1) / CH;
    auto place = [&](int c) { return (a.back ? chunks - 1 - c : c) * CH; };
    Fetch<BF16, DK, NT, VEC> fk(a.k, s, g, h, a.dk, place(0));
    Fetch<BF16, DV, NT, VEC> fv(a.v, s, g, h, a.dv, place(0));
    uint32_t decay = 0;
    RowPointer rate(s.g, s.g_row, s.g_head, s, g, h, place(0) + l, a.back ? -CH : CH);
    auto ask = [&](int p) {
        if (wave == 0) decay = raw_decay(s, rate, g.n, l < CH), rate.next(a.back ? -CH : CH);
        fk.load(a.k, s, g, h, p, a.dk, !a.back);
        fv.load(a.v, s, g, h, p, a.dv, !a.back);
    };
    double sum = 0.0;
    ask(place(0));
    if (wave == 0) sum = chunk_decays(s, decay, &lds.d[0], a.scale);
    for (int c = 0, now = 0; c < chunks; ++c, now ^= 1) {
        __syncthreads();
        fk.store(tk, a.dk), fv.store(tv, a.dv);
        __syncthreads();
        if (c + 1 < chunks) ask(place(c + 1));
        frag of[C * (CH / KS)];
#pragma unroll
        for (int ct = 0; ct < C; ++ct)
#pragma unroll
            for (int k = 0; k < CH / KS; ++k) of[ct * (CH / KS) + k] = tv.columns(l, k * KS, col0 + ct * 16);
        W::template add<TERMS, CH>(st, of, tk, lds.d[now], a.back ? lds.d[now].since : lds.d[now].left);
        if (wave == 0 && c + 1 < chunks) sum += chunk_decays(s, decay, &lds.d[now ^ 1], a.scale);
    }
    W::save(st, a.bound + (i * s.H + h) * (long long)(a.dk * a.dv), a.st.sk, a.st.sv, a.dk, a.dv, col0);
    if (threadIdx.x == 0) a.decay[i * s.H + h] = __builtin_amdgcn_exp2f((float)sum);
}

// Along the boundaries of a sequence, in place: the state in front of each segment (back: the gradient of it). A thread has W adjacent elements; a block of each
// sequence that has boundaries does its share of them, found by the sequence's number or, where there are fewer, by its first boundary's. Eight states are on their way
// at once (64 boundaries of 8 heads of 64 x 128: 16.8 us, sixteen 15.8; 32 of 16 heads of 128 x 128: 13.6 and 17.6).
template <int W> __global__ void __launch_bounds__(256) scan_kernel(const ScanArgs a) {
    const Shape& s = a.s;
    const int h = blockIdx.x % (unsigned)s.H;
    const long long which = blockIdx.x / (unsigned)s.H;
    int seq, lo, hi;
    if (a.by_sequence) {
        seq = (int)which - 1, lo = edge_of(s, which), hi = edge_of(s, which + 1);
        if ((long long)hi - lo <= s.L) return;
    } else {
        const Segment g = boundary(s, 1 + which);
        if (g.n == 0 || g.p0 != s.L) return;
        seq = g.seq, lo = g.lo, hi = g.hi;
    }
    const int at = (blockIdx.y * 256 + threadIdx.x) * W;
    if (at >= a.n) return;
    typedef float vec __attribute__((ext_vector_type(W)));
    const long long m = ((long long)hi - lo - 1) / s.L, first = lo / s.L + 1;        // the sequence's boundaries, first, first + 1 .. (its rows lie L apart)
    const long long way = a.back ? -1 : 1, begin = a.back ? first + m - 1 : first;
    vec now = {};
    if (a.edge && seq >= 0 && seq < s.S) now = *(const vec*)(a.edge + ((long long)seq * s.H + h) * a.n + at);
    constexpr int AHEAD = 8;
    vec add[AHEAD];
    float dec[AHEAD];
    auto ask = [&](long long j) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const long long b = (begin + way * (j + e < m ? j + e : m - 1)) * s.H + h;
            add[e] = *(const vec*)(a.bound + b * a.n + at);
            dec[e] = a.decay[b];
        }
    };
    ask(0);
    for (long long j = 0; j < m; j += AHEAD) {
        vec out[AHEAD];
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) out[e] = now = dec[e] * now + add[e];       // (beyond the last boundary: not kept)
        if (j + AHEAD < m) ask(j + AHEAD);
#pragma unroll
        for (int e = 0; e < AHEAD; ++e)
            if (j + e < m) *(vec*)(a.bound + ((begin + way * (j + e)) * s.H + h) * a.n + at) = out[e];
    }
}

// ---- gradients of keys, values and decays ---------------------------------------------------------------------------------------------
// The chunks of a segment from the last to the first. Half of the waves have dv, the other half dk: a state in registers for each, and either sees the other's scores.
// No unit is full: vector instructions take half of the SIMDs' cycles, the products 0.13, and waves wait for 0.39 of theirs, which two blocks a CU do not hide: 131072 rows of 16 heads of 64
// in bf16 600 us (351 as loads and stores alone; when it took 634, the log decays' gradient was 160 of them). A third block a CU has no registers (168 of the 223: it spills), twice the waves of half the
// columns took as long.
// One block has both gradients, or each has a launch: where keys are wide, a block of both has no room for a second one on its CU, and dk's waves have more to do than
// dv's. Backward of 65536 rows in sequences of 266, 16 heads of 128 x 128: 1503 us together, 1221 apart; 128 x 64 893 and 852; 64 x 128 (20011 rows of 8 heads, these
// kernels) 100 and 104.
constexpr bool back_apart(int dk, int) { return dk == 128; }
constexpr int back_threads(int dk, int dv) { return back_apart(dk, dv) ? 256 : (dk > dv ? dk : dv) * 4; }
enum { BOTH, VALUES, KEYS };         // what a block has: dv and dk, or one of them (the decays' gradient goes with dk)
template <bool BF16, int DK, int DV, int ROLE, bool DG> struct BackLds {
    static constexpr int CH = chunk_rows(BF16);
    char q[Tile<BF16, DK>::BYTES], k[ROLE != KEYS || DG ? Tile<BF16, DK>::BYTES : 16], v[ROLE != VALUES ? Tile<BF16, DV>::BYTES : 16], o[Tile<BF16, DV>::BYTES];
    char a[ROLE != KEYS ? Tile<BF16, CH>::BYTES : 16], b[ROLE != VALUES ? Tile<BF16, CH>::BYTES : 16];
    Decays<CH> d[2];
    alignas(16) float reads[DG ? CH / 16 : 1][CH];            // (written four at a time)
    float given[DG ? CH / 16 : 1][CH], w[DG ? 4 : 1][CH];
    double sum[2][DG ? 8 : 1];
    double size[2][DG ? CH : 1];     // what rows' terms may be off by goes with (one decay a head)
};
static_assert(__builtin_offsetof(BackLds<true, 64, 64, BOTH, true>, reads) % 16 == 0, "rows of four");
// TERMS: of the state that the keys' gradient and with it that of the log decays come from; VTERMS: of the values', which may be the initial states' gradient. The first
// wave also has the chunk's decays, the second one the log decays' gradient: where that is wanted, the keys' waves have more to do.
template <bool BF16, int DK, int DV, int ROLE, int TERMS, int VTERMS, bool DG, bool VEC>
__global__ void __launch_bounds__(back_threads(DK, DV), 2) back_kernel(const BackArgs a) {
    typedef Op<BF16> O;
    typedef typename O::frag frag;
    constexpr int NT = back_threads(DK, DV), NW = NT / 64, HW = ROLE == BOTH ? NW / 2 : NW, KS = O::KS, CH = O::CH, CV = DV / 16 / HW, CK = DK / 16 / HW, C = CV > CK ? CV : CK;
    typedef Role<BF16, DK, CV, false> V;                            // dS[key][values]: dv
    typedef Role<BF16, DV, CK, false> K;                            // dS[value][keys]: dk
    static_assert(V::SR * CV == K::SR * CK, "either role has as much of the state");
    __shared__ __attribute__((aligned(256))) BackLds<BF16, DK, DV, ROLE, DG> lds;
    const Tile<BF16, DK> tq{lds.q}, tk{lds.k};
    const Tile<BF16, DV> tv{lds.v}, to{lds.o};
    const Tile<BF16, CH> ta{lds.a}, tb{lds.b};
    const Shape& s = a.s;
    const int h = blockIdx.x % (unsigned)s.H, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
    const long long slot = blockIdx.x / (unsigned)s.H;
    const Segment g = segment_at(s, slot);
    const int n = a.dk * a.dv, mine = wave % HW;
    const bool states = g.real(s), values = ROLE == BOTH ? wave < HW : ROLE == VALUES;
    const int col0 = mine * 16 * (values ? CV : CK);
    if (g.n == 0) {
        if (DG && a.dg_part && threadIdx.x == 0) a.dg_part[slot * s.H + h] = 0.0;
        // an empty sequence's state goes through
        if (ROLE != KEYS && a.dinitial && states && g.p0 == 0 && g.hi <= g.lo)
            for (int e = threadIdx.x; e < n; e += NT) a.dinitial[((long long)g.seq * s.H + h) * n + e] = a.dstate ? a.dstate[((long long)g.seq * s.H + h) * n + e] : 0.f;
        return;
    }
    const int end = (g.n - 1) / CH * CH;
    Fetch<BF16, DK, NT, VEC> fq(a.q, s, g, h, a.dk, end), fk(a.k, s, g, h, a.dk, end);
    Fetch<BF16, DV, NT, VEC> fv(a.v, s, g, h, a.dv, end), fo(a.o, s, g, h, a.dv, end);
    Drain<BF16, DK, NT, VEC> out_k(a.dk_out, s, g, h, a.dk, end);
    Drain<BF16, DV, NT, VEC> out_v(a.dv_out, s, g, h, a.dv, end);
    uint32_t decay = 0;
    float u = 0.f;
    RowPointer rate(s.g, s.g_row, s.g_head, s, g, h, end + l, CH), us(a.u, 4, 4ll * s.T, s, g, h, end + l, CH);
    const int de = a.dg_bf16 ? 2 : 4;
    RowPointer dgs(a.dg, (long long)s.H * de, de, s, g, h, end + l, CH);
    auto ask = [&](int p) {
        if (wave == 0) decay = raw_decay(s, rate, g.n, l < CH), rate.back(CH);
        if constexpr (DG)
            if (wave == 1) u = l < CH && us.place < g.n ? *(const float*)us.p : 0.f, us.back(CH);
        fq.load(a.q, s, g, h, p, a.dk, false);
        if constexpr (ROLE != KEYS || DG) fk.load(a.k, s, g, h, p, a.dk, false);
        if constexpr (ROLE != VALUES) fv.load(a.v, s, g, h, p, a.dv, false);
        fo.load(a.o, s, g, h, p, a.dv, false);
    };
    auto take = [&] {
        if constexpr (ROLE != VALUES) out_k.take(ROLE == BOTH ? tk : tq);
        if constexpr (ROLE != KEYS) out_v.take(ROLE == BOTH ? tv : to);
    };
    auto give = [&](int p) {
        if constexpr (ROLE != VALUES) out_k.give(s, g, p, a.dk, false);
        if constexpr (ROLE != KEYS) out_v.give(s, g, p, a.dv, false);
    };
    ask(end);
    f32x4 st[V::SR * CV];
#pragma unroll
    for (int t = 0; t < V::SR * CV; ++t) st[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const bool last = g.last();
    const float* const start = g.p0 > 0 ? a.bound : states ? a.initial : nullptr;        // what the segment begins with, where the log decays' gradient looks at it
    const bool keep = (a.dinitial && states && g.p0 == 0) || (DG && a.dg_part && start && !a.dg_bf16);
    const float *from = !last ? a.gbound : states ? a.dstate : nullptr, *with = !last ? a.bound : states ? a.state : nullptr;
    const bool weigh = DG && a.dg_part && !a.dg_bf16;
    double cross = 0.0, squares = 0.0;                        // <S, dS> behind the rows that were done; of its products
    if (from) {
        const long long at = ((!last ? g.bound(s) + 1 : g.seq) * s.H + h) * (long long)n;       // (the next boundary lies L rows on; of a sequence's first segment (lo + L) / L)
        if (values) V::load(st, from + at, a.dv, 1, a.dk, a.dv, col0);
        else K::load(st, from + at, 1, a.dv, a.dv, a.dk, col0);
        if constexpr (DG)
            if (with)
                for (int e = threadIdx.x; e < n; e += NT) {
                    const double x = (double)from[at + e] * (double)with[at + e];
                    cross += x, squares = fma(x, x, squares);
                }
    }
    if constexpr (DG) {
#pragma unroll
        for (int m = 1; m < 64; m *= 2) cross += __shfl_xor(cross, m), squares += __shfl_xor(squares, m);
        if (l == 0) lds.sum[0][wave] = cross, lds.sum[1][wave] = squares;
        __syncthreads();
        cross = squares = 0.0;
#pragma unroll
        for (int w = 0; w < NW; ++w) cross += lds.sum[0][w], squares += lds.sum[1][w];
        if (wave == 1 && l < CH) lds.size[0][l] = l ? 0.0 : g.n * squares, lds.size[1][l] = l ? 0.0 : squares;
    }
    double total = 0.0;
    if (wave == 0) chunk_decays(s, decay, &lds.d[0], a.scale);
    for (int p = end, now = 0; p >= 0; p -= CH, now ^= 1) {
        const Decays<CH>& d = lds.d[now];
        __syncthreads();
        if (p < end) take();
        fq.store(tq, a.dk), fo.store(to, a.dv);
        if constexpr (ROLE != KEYS || DG) fk.store(tk, a.dk);
        if constexpr (ROLE != VALUES) fv.store(tv, a.dv);
        if (p < end) give(p + CH);
        const float u_now = u;
        __syncthreads();
        if (p > 0) ask(p - CH);
        const bool half = halves(BF16, DK, DV) && g.n - p <= CH / 2;
        for (int t = wave; t < O::SCORES; t += NW) {
            int it, jt;
            const int l = this_lane(), lr = l & 15, lg = l >> 4;
            O::score(t, false, it, jt);
            const int j = jt * 16 + lr, i = it * 16 + lg * 4;
            if (it * 16 >= (half ? CH / 2 : CH)) continue;    // (nobody looks at it)
            if (jt > it) {
                const f32x4 none = {0.f, 0.f, 0.f, 0.f};
                if constexpr (ROLE != KEYS) ta.put_quad(j, i, none);
                if constexpr (ROLE != VALUES) tb.put_quad(j, i, none);
                if constexpr (DG) {
                    if (lg == 0) lds.given[it][j] = 0.f;
                    if (lr == 0) *(f32x4*)(lds.reads[jt] + i) = none;
                }
                continue;
            }
            f32x4 ca = {0.f, 0.f, 0.f, 0.f}, cb = {0.f, 0.f, 0.f, 0.f}, both, w;
            if constexpr (ROLE != KEYS || DG)
#pragma unroll
                for (int k = 0; k < DK; k += KS) ca = O::mma(tq.rows(l, it * 16, k), tk.rows(l, jt * 16, k), ca);
            if constexpr (ROLE != VALUES)
#pragma unroll
                for (int k = 0; k < DV; k += KS) cb = O::mma(to.rows(l, it * 16, k), tv.rows(l, jt * 16, k), cb);
            f32x4 e = *(const f32x4*)(d.hi + i) - d.hi[j];
            if constexpr (fine<BF16, TERMS>()) e += *(const f32x4*)(d.lo + i) - d.lo[j];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = __builtin_amdgcn_exp2f(e[r]) * a.scale;
            ca *= w;
            both = ca * cb;
            cb *= w;
            if (jt == it) {                                   // (on the diagonal: what lies above it, and of the products of scores it, too)
                asm volatile("");                             // (a branch: three tiles of ten take it)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    ca[r] = i + r < j ? 0.f : ca[r];
                    cb[r] = i + r < j ? 0.f : cb[r];
                    both[r] = i + r <= j ? 0.f : both[r];
                }
            }
            if constexpr (ROLE != KEYS) ta.put_quad(j, i, ca);
            if constexpr (ROLE != VALUES) tb.put_quad(j, i, cb);
            if constexpr (DG) {
                const float given = lane_sum4((both[0] + both[1]) + (both[2] + both[3]));
                if (lg == 0) lds.given[it][j] = given;
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = lane_sum16(both[r]);
                if (lr == 0) *(f32x4*)(lds.reads[jt] + i) = v;
            }
        }
        __syncthreads();
        f32x4 res[C * (CH / 16)];
        frag of[C * (CH / KS) > C * (CH / 16) ? C * (CH / KS) : C * (CH / 16)];
        auto read = [&](auto rows) {
            if (values) V::template read<2, false, rows.value>(st, res, of, tk, to, ta, tk, d, col0, nullptr, p < end || from);
            else K::template read<DG ? TERMS : 2, DG, rows.value>(st, res, of, tv, tq, tb, tk, d, col0, DG ? lds.w[mine] : nullptr, p < end || from);
        };
        if (half) read(Rows_<CH / 2>{}); else read(Rows_<CH>{});
        // The results take the place of keys and values, once these have been read; where a block has one of them, that of its own columns, which each wave has in of.
        if constexpr (ROLE == BOTH) __syncthreads();
        auto put = [&](auto rows) {
            if (values) V::template put<rows.value>(res, ROLE == BOTH ? tv : to, col0);
            else K::template put<rows.value>(res, ROLE == BOTH ? tk : tq, col0);
        };
        if (half) put(Rows_<CH / 2>{}); else put(Rows_<CH>{});
        if constexpr (ROLE != BOTH && DG) __syncthreads();
        if constexpr (DG)
            if (wave == 1) {
                float e = u_now, size = fabsf(u_now);
                auto term = [&](float x) { e += x, size += fabsf(x); };
                if (l < CH) {
#pragma unroll
                    for (int t = 0; t < CH / 16; ++t) {
                        if (t * 16 < O::reads_to(l >> 4)) term(lds.reads[t][l]);
                        if (t * 16 >= O::read_from(l >> 4) && (t < CH / 32 || !half)) term(-lds.given[t][l]);
                    }
#pragma unroll
                    for (int w = 0; w < HW; ++w) term(-lds.w[w][l]);
                }
                if (weigh && l < CH && p + l < g.n) {
                    const double q = (double)size * size;
                    lds.size[0][l] += q * (p + l + 1), lds.size[1][l] += q;
                }
                const double mine = l < (half ? CH / 2 : CH) ? e : 0.f, upto = running_sum<CH>(mine), all = __shfl(upto, CH - 1), dg = (all - upto) + mine + cross;
                cross += all;
                if (l < CH && p + l < g.n) {
                    total += dg;
                    if (a.dg) {
                        if (a.dg_bf16) *(uint16_t*)dgs.p = f32_to_bf16((float)dg);
                        else *(float*)dgs.p = (float)dg;
                    }
                }
                dgs.back(CH);
            }
        auto add = [&](auto rows) {
            if (values) V::template add<VTERMS, rows.value>(st, of, tq, d, d.since);
            else K::template add<TERMS, rows.value>(st, of, to, d, d.since);
        };
        if (p > 0 || keep) {
            if (half) add(Rows_<CH / 2>{}); else add(Rows_<CH>{});
        }
        if (wave == 0 && p > 0) chunk_decays(s, decay, &lds.d[now ^ 1], a.scale);
    }
    __syncthreads();
    take();
    give(0);
    if constexpr (DG)
        if (a.dg_part) {
            // What the rows' sum must come to is known as well, <S, dS> in front of the segment. What it is off by has come row by row: an error of row t is t + 1 times in the
            // rows' sum, one of <S, dS> behind the segment g.n times, one of that in front of it not at all. Errors being independent and going with the sizes of the
            // terms, the part of the difference that the rows' sum has is on the average the squares' sum with these numbers over the squares' sum (the products in front
            // sixteen times: the gradient of a state has the errors of all rows behind it; without them a state 100 times as large made it three times worse). Errors of a segment
            // of 2048 rows (64 x 64, 32 heads, relative to the 2-norm of the rows' gradients) without and with it: rows of one size, decay 0.5 1.1e-4 and 5.1e-5, 0.97
            // 5.4e-5 and 2.4e-5; an initial state 1000 times as large 5.1e-6 and 2.4e-6 both; keys that grow by e^7 1.8e-4 and 8.8e-6. A sum in bf16 is rounded by more.
            double known = 0.0;
            squares = 0.0;
            if (start && weigh && !values) K::dot(st, start + ((g.p0 > 0 ? g.bound(s) : g.seq) * s.H + h) * (long long)n, 1, a.dv, a.dv, a.dk, col0, known, squares);
            double rows = l < CH ? lds.size[0][l] : 0.0, all = l < CH ? lds.size[1][l] : 0.0;          // (the second wave's)
#pragma unroll
            for (int m = 1; m < 64; m *= 2) {
                known += __shfl_xor(known, m), squares += __shfl_xor(squares, m), total += __shfl_xor(total, m);
                rows += __shfl_xor(rows, m), all += __shfl_xor(all, m);
            }
            if (l == 0) lds.sum[0][wave] = known, lds.sum[1][wave] = squares;
            __syncthreads();
            known = 0.0;
#pragma unroll
            for (int w = NW - HW; w < NW; ++w) known += lds.sum[0][w], all += 16.0 * lds.sum[1][w];
            const double share = rows / all;                  // (NaN without terms, or with infinite ones)
            if (wave == 1 && l == 0) a.dg_part[slot * s.H + h] = weigh && share > 0.0 ? total - share * (cross - known) : total;
        }
    if (a.dinitial && states && g.p0 == 0 && values) V::save(st, a.dinitial + ((long long)g.seq * s.H + h) * n, a.dv, 1, a.dk, a.dv, col0);
}

// One decay a head: the sum of the segments' sums, in a fixed order.
__global__ void __launch_bounds__(256) sum_kernel(const double* part, long long slots, int H, void* out, int bf16) {
    __shared__ double lds[256];
    const int h = blockIdx.x;
    double v = 0.0;
    for (long long i = threadIdx.x; i < slots; i += 256) v += part[i * H + h];
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int m = 128; m > 0; m >>= 1) {
        if ((int)threadIdx.x < m) lds[threadIdx.x] += lds[threadIdx.x + m];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (bf16) ((uint16_t*)out)[h] = f32_to_bf16((float)lds[0]);
        else ((float*)out)[h] = (float)lds[0];
    }
}

// ---- one token of each sequence -------------------------------------------------------------------------------------------------------
// A block has COLS columns of one head's state of one row: COLS / W lanes with W adjacent columns each, and 256 * W / COLS such groups with every that many key's
// row. Bound by memory, the state in and out: a thread asks for eight rows before it uses the first (250 sequences of 16 x 128 x 128: four 96 us, eight 96, sixteen
// 136). ONCE: past the caches, for more states than they hold (89 us). A row whose slot an earlier row names is done by that row's
// block, behind it, so that they are consecutive tokens of one sequence.
__device__ __forceinline__ float element(const char* p, int i, int bf16) { return bf16 ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i]; }

template <int COLS, int W, bool ONCE> __global__ void __launch_bounds__(256) step_kernel(const StepArgs a) {
    constexpr int LR = COLS / W, G = 256 / LR, AHEAD = 8;
    typedef float vec __attribute__((ext_vector_type(W)));
    __shared__ __attribute__((aligned(16))) float part[G][COLS];      // (written W at a time)
    __shared__ float keys[2][128];                            // k, q
    __shared__ int first;
    const int h = blockIdx.x % (unsigned)a.H, b = blockIdx.x / (unsigned)a.H, col0 = blockIdx.y * COLS, lane = threadIdx.x % LR, gk = threadIdx.x / LR;
    const int c = col0 + lane * W, e = a.bf16 ? 2 : 4;
    const bool mine = c < a.dv;                               // (W divides dv)
    const long long slot = a.slots ? a.slots[b] : b;
    auto write = [&](int row, int column, float v) {
        char* const at = a.o + ((long long)row * a.H + h) * a.dv * e;
        if (a.bf16) ((uint16_t*)at)[column] = f32_to_bf16(v);
        else ((float*)at)[column] = v;
    };
    if (slot < 0 || slot >= a.N) {
        if ((int)threadIdx.x < COLS && col0 + (int)threadIdx.x < a.dv) write(b, col0 + threadIdx.x, 0.f);
        return;
    }
    const long long at = (slot * a.H + h) * (long long)a.dk * a.dv + c;
    const float* from = a.state + at;
    float* const to = a.out_state + at;
    vec old[AHEAD];
    auto ask = [&](const float* p, int i0) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * G;
            const vec* const x = (const vec*)(p + (long long)i * a.dv);
            if (mine && i < a.dk) old[j] = ONCE ? __builtin_nontemporal_load(x) : *x;
        }
    };
    ask(from, gk);
    if (a.slots) {                                            // an earlier row of this slot does this one, too
        bool earlier = false;
        int next = a.B;
        for (int r0 = threadIdx.x; r0 < a.B; r0 += 8 * 256) { // (all rows: those behind, for the next one)
            int at[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) at[j] = r0 + j * 256 < a.B ? a.slots[r0 + j * 256] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = r0 + j * 256;
                earlier = earlier || (at[j] == (int)slot && r < b);
                if (at[j] == (int)slot && r > b && r < next) next = r;
            }
        }
        if (threadIdx.x == 0) first = a.B;
        if (__syncthreads_or(earlier)) return;
        if (next < a.B) atomicMin(&first, next);              // (in the LDS; the least of them whatever their order)
    }
    int row = b;
    while (true) {
        const char *q = a.q.p + row * a.q.row + h * a.q.head, *k = a.k.p + row * a.k.row + h * a.k.head, *v = a.v.p + row * a.v.row + h * a.v.head;
        for (int i = threadIdx.x; i < 2 * a.dk; i += 256) keys[i >= a.dk][i >= a.dk ? i - a.dk : i] = i >= a.dk ? element(q, i - a.dk, a.bf16) : element(k, i, a.bf16);
        const float dec = __builtin_amdgcn_exp2f(element(a.g + row * a.g_row + h * a.g_head, 0, a.g_bf16) * 1.44269504088896341f);
        vec vc = {}, sum = {};
        if (mine)
#pragma unroll
            for (int w = 0; w < W; ++w) vc[w] = element(v, c + w, a.bf16);
        __syncthreads();
        for (int i0 = gk; i0 < a.dk; i0 += AHEAD * G) {
            vec now[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = i0 + j * G;
                if (mine && i < a.dk) now[j] = dec * old[j] + keys[0][i] * vc, sum += keys[1][i] * now[j];
            }
            if (i0 + AHEAD * G < a.dk) ask(from, i0 + AHEAD * G);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = i0 + j * G;
                vec* const x = (vec*)(to + (long long)i * a.dv);
                if (mine && i < a.dk) {
                    if constexpr (ONCE) __builtin_nontemporal_store(now[j], x); else *x = now[j];
                }
            }
        }
        *(vec*)&part[gk][lane * W] = sum;
        __syncthreads();
        if ((int)threadIdx.x < COLS && col0 + (int)threadIdx.x < a.dv) {
            float o = 0.f;
#pragma unroll 8
            for (int i = 0; i < G; ++i) o += part[i][threadIdx.x];
            write(row, col0 + threadIdx.x, o * a.scale);
        }
        if (!a.slots) return;
        int next = row == b ? first : a.B;                    // the next row of the slot
        for (int r0 = row + 1; row != b && r0 < a.B && next == a.B; r0 += 256) {
            const int r = r0 + threadIdx.x;
            const bool same = r < a.B && a.slots[r] == (int)slot;
            __syncthreads();
            if (threadIdx.x == 0) first = a.B;
            __syncthreads();
            if (same) atomicMin(&first, r);
            __syncthreads();
            next = first;
        }
        if (next >= a.B) return;
        row = next;
        from = to;                                            // (each thread reads what it wrote itself)
        ask(from, gk);
        __syncthreads();
    }
}

}  // namespace la
}  // namespace nplm
