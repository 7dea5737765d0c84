// Kernels of the layer norm (include/nplm_layernorm.h).
//
// G lanes have the channels of one head of a row in registers (norm_rows.h): read once, statistics as sums over the G lanes, written once. A group
// keeps its head and goes through many rows with that head's parameters, and in the backward with their gradients, in registers. A block has R = 256 / G
// groups (one where G is larger): the heads of R / heads rows, or, where a row has more heads than that, R of them (blockIdx.y says which).
// The backward forms the statistics again: they cost less than a word of 8 bytes a head, written and read.
#pragma once
#include "norm_rows.h"

namespace nplm {
namespace ln {

using rn::group_sum;
using rn::load_param;
using rn::Slice;
using rn::statistics;

struct Args {
    const char *x, *gate, *dy;
    long long xs, gs, ds;             // row strides in bytes
    const void *weight, *bias;
    char *y, *dgate;                  // y: dx in the backward
    float* partial;                   // [2][blocks][columns]
    float eps;
    int T, C, heads, n, w_bf16, rms, shared, want;
};

// Where a group of lanes works: its head, its first row and how far apart its rows are.
template <int G> struct Place {
    int head, row, step;
    bool there;
    __device__ __forceinline__ Place(const Args& a) {
        constexpr int R = G > 256 ? 1 : 256 / G;
        const int group = threadIdx.x / G, rows = a.heads < R ? R / a.heads : 1;
        head = a.heads < R ? group % a.heads : blockIdx.y * R + group;
        row = blockIdx.x * rows + (a.heads < R ? group / a.heads : 0);
        step = gridDim.x * rows;
        there = head < a.heads && (a.heads >= R || group < rows * a.heads);
        if (!there) head = 0;
    }
};

template <bool BF16, int VEC, int G, int PL>
__global__ void __launch_bounds__(G > 256 ? G : 256) fwd_kernel(const Args p) {
    constexpr int E = BF16 ? 2 : 4;
    __shared__ float lds[G > 64 ? 16 : 1];
    const int g = threadIdx.x % G;
    const Place<G> at(p);
    const long long off = (long long)at.head * p.n;
    Slice<BF16, VEC, PL> xv, gv;
    auto ask = [&](long long t) {
        const int n = at.there && t < p.T ? p.n : 0;
        const size_t r = t < p.T ? t : 0;
        xv.template load<G>(p.x + r * p.xs + off * E, g, n);
        if (p.gate) gv.template load<G>(p.gate + r * p.gs + off * E, g, n);
    };
    ask(at.row);
    float w[PL], b[PL];
    const char* const pw = (const char*)p.weight + (p.shared ? 0 : off) * (p.w_bf16 ? 2 : 4);
    const char* const pb = (const char*)p.bias + (p.shared ? 0 : off) * (p.w_bf16 ? 2 : 4);
    load_param<VEC, G, PL>(w, p.weight ? pw : nullptr, p.w_bf16, g, p.n, 1.f);
    load_param<VEC, G, PL>(b, p.bias ? pb : nullptr, p.w_bf16, g, p.n, 0.f);
    // (all groups of a block as often as its first one: they meet in group_sum)
    for (long long t0 = (long long)blockIdx.x * (at.step / gridDim.x), t = at.row; t0 < p.T; t0 += at.step, t += at.step) {
        float v[PL], m, r;
        xv.to_f32(v);
        statistics<VEC, G, PL>(v, g, p.n, p.rms, p.eps, m, r, lds);
#pragma unroll
        for (int j = 0; j < PL; ++j) v[j] = fmaf((v[j] - m) * r, w[j], b[j]);
        if (p.gate) {
            float ga[PL];
            gv.to_f32(ga);
#pragma unroll
            for (int j = 0; j < PL; ++j) v[j] *= ga[j] * sigmoid_f32(ga[j]);
        }
        if (t0 + at.step < p.T) ask(t + at.step);
        Slice<BF16, VEC, PL> out;
        out.from_f32(v);
        if (at.there && t < p.T) out.template store<G>(p.y + ((size_t)t * p.C + off) * E, g, p.n);
    }
}

template <bool BF16, int VEC, int G, int PL>
__global__ void __launch_bounds__(G > 256 ? G : 256) bwd_kernel(const Args p) {
    constexpr int NT = G > 256 ? G : 256, R = NT / G, E = BF16 ? 2 : 4;
    __shared__ float lds[G > 64 ? 32 : 1];
    __shared__ float part[R > 1 ? R : 1][R > 1 ? G * PL : 1];
    const int g = threadIdx.x % G;
    const Place<G> at(p);
    const long long off = (long long)at.head * p.n;
    Slice<BF16, VEC, PL> xv, gv, dv;
    auto ask = [&](long long t) {                         // (lanes without a row have zeros, which add nothing; a 0 times what another row holds may be NaN)
        const int n = at.there && t < p.T ? p.n : 0;
        const size_t r = t < p.T ? t : 0;
        xv.template load<G>(p.x + r * p.xs + off * E, g, n);
        if (p.gate) gv.template load<G>(p.gate + r * p.gs + off * E, g, n);
        dv.template load<G>(p.dy + r * p.ds + off * E, g, n);
    };
    ask(at.row);
    float w[PL], b[PL];
    const char* const pw = (const char*)p.weight + (p.shared ? 0 : off) * (p.w_bf16 ? 2 : 4);
    const char* const pb = (const char*)p.bias + (p.shared ? 0 : off) * (p.w_bf16 ? 2 : 4);
    load_param<VEC, G, PL>(w, p.weight ? pw : nullptr, p.w_bf16, g, p.n, 1.f);
    load_param<VEC, G, PL>(b, p.bias && p.gate ? pb : nullptr, p.w_bf16, g, p.n, 0.f);
    float sum[2][PL] = {};
    const float inv = 1.f / p.n;
    for (long long t0 = (long long)blockIdx.x * (at.step / gridDim.x), t = at.row; t0 < p.T; t0 += at.step, t += at.step) {
        float v[PL], d[PL], ga[PL], m, r;
        const bool real = at.there && t < p.T;
        xv.to_f32(v);
        dv.to_f32(d);
        if (p.gate) gv.to_f32(ga);
        if (t0 + at.step < p.T) ask(t + at.step);
        statistics<VEC, G, PL>(v, g, p.n, p.rms, p.eps, m, r, lds);
#pragma unroll
        for (int j = 0; j < PL; ++j) v[j] = real && ((j / VEC) * G + g) * VEC < p.n ? (v[j] - m) * r : 0.f;
        if (p.gate) {
            float dg[PL];
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                const float sg = sigmoid_f32(ga[j]);
                dg[j] = d[j] * fmaf(v[j], w[j], b[j]) * sg * fmaf(ga[j], 1.f - sg, 1.f);
                d[j] *= ga[j] * sg;
            }
            Slice<BF16, VEC, PL> out;
            out.from_f32(dg);
            if (real) out.template store<G>(p.dgate + ((size_t)t * p.C + off) * E, g, p.n);
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < PL; ++j) {
            sum[0][j] = fmaf(d[j], v[j], sum[0][j]);
            sum[1][j] += d[j];
            d[j] *= w[j];
            s[0] += d[j];                                 // (zero beyond n, as v is)
            s[1] = fmaf(d[j], v[j], s[1]);
        }
        group_sum<G, 2>(s, lds);
        const float m0 = p.rms ? 0.f : s[0] * inv, m1 = s[1] * inv;
#pragma unroll
        for (int j = 0; j < PL; ++j) d[j] = r * (d[j] - m0 - v[j] * m1);
        Slice<BF16, VEC, PL> out;
        out.from_f32(d);
        if (real) out.template store<G>(p.y + ((size_t)t * p.C + off) * E, g, p.n);
    }
    // the block's sums: of one weight for all heads over all groups, else over the groups of each head
    const int columns = p.shared ? p.n : p.C, blocks = p.shared ? gridDim.x * gridDim.y : gridDim.x, block = p.shared ? blockIdx.y * gridDim.x + blockIdx.x : blockIdx.x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!(p.want >> i & 1)) continue;
        float* to = p.partial + ((size_t)i * blocks + block) * columns;
        if constexpr (R > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PL; ++j) part[threadIdx.x / G][((j / VEC) * G + g) * VEC + j % VEC] = sum[i][j];
            __syncthreads();
            const int apart = p.shared ? 1 : p.heads < R ? p.heads : R;     // groups of the same column lie so far apart
            const int first = p.heads < R ? 0 : blockIdx.y * R;             // the block's first head
            for (int u = threadIdx.x; u < apart * p.n; u += NT) {
                const int h = u / p.n, c = u - h * p.n;
                if (!p.shared && first + h >= p.heads) continue;
                float s = 0.f;
                for (int r = h; r < R; r += apart) s += part[r][c];         // (groups without a head have zeros)
                to[p.shared ? c : (first + h) * p.n + c] = s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                const int c = ((j / VEC) * G + g) * VEC + j % VEC;
                if (c < p.n) to[(p.shared ? 0 : at.head * p.n) + c] = sum[i][j];
            }
        }
    }
}

// Adds up the blocks' sums, in fp64: 16 columns a block, each of its 64 groups of lanes every 64th block's sums, eight loads at a time, then the groups'.
__global__ void __launch_bounds__(1024) sum_kernel(const float* partial, void* out0, void* out1, int blocks, int columns, int bf16) {
    __shared__ double part[64][16];
    const int i = blockIdx.y, j = threadIdx.x / 16, lane = threadIdx.x % 16, c = blockIdx.x * 16 + lane;
    void* const out = i ? out1 : out0;
    if (!out) return;
    double s = 0;
    if (c < columns) {
        const float* at = partial + (size_t)i * blocks * columns + c;
        int b = j;
        for (; b + 7 * 64 < blocks; b += 8 * 64) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = at[(size_t)(b + u * 64) * columns];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; b < blocks; b += 64) s += at[(size_t)b * columns];
    }
    part[j][lane] = s;
    __syncthreads();
    if (j || c >= columns) return;
    s = 0;
#pragma unroll 8
    for (int w = 0; w < 64; ++w) s += part[w][lane];
    if (bf16) ((uint16_t*)out)[c] = f32_to_bf16((float)s);
    else ((float*)out)[c] = (float)s;
}

}  // namespace ln
}  // namespace nplm
