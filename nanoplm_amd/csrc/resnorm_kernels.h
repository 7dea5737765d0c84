// Kernels of the residual norm (include/nplm_resnorm.h).
//
// G lanes have a row (G a power of two, 8 to 1024: part of a wave, a wave or a block of waves) and each of them PL of its channels in
// registers, in vectors of VEC adjacent ones, so that a row is read once, its statistics are sums over the G lanes, and it is written once.
// A group goes through many rows with the parameters in its registers; in the backward it keeps the parameters' gradients there too.
#pragma once
#include "norm_rows.h"

namespace nplm {
namespace rn {

constexpr int kParams = 5;       // post_weight, post_bias, scale, pre_weight, pre_bias

struct FwdArgs {
    const char *u, *gate, *residual;
    long long us, gs, rs;             // row strides in bytes
    const void* par[kParams];
    char *out, *normed;
    float* stats;
    float eps;
    int T, C, w_bf16, rms;
};
struct BwdArgs {
    const char *u, *gate, *residual, *dout, *dnormed;
    long long us, gs, rs, os, ns;
    const float* stats;
    const void* par[kParams];
    char *du, *dgate, *dresidual;
    float* partial;                   // [blocks][kParams][C]
    int T, C, w_bf16, rms, want;      // want: bit i, the gradient of parameter i
};

// Bound by memory: a row's 5 or so words a channel are read and written once, with some 20 operations between. T=131072, C=1024 with gate, both norms and a scale:
// bf16 261 us (5.1 TB/s; a copy of 256 MiB here reaches 5.6, with nt hints 6.2), T=50021, C=768, bf16 branches on an fp32 stream 111 us (4.8 TB/s), T=5003, C=1001, fp32 19 us.
// A row is asked for before the one in front of it is written, the first one before the parameters: 8 rows of 2048 9.2 -> 4.3 us, with the parameters in vectors.
template <bool ABF, bool SBF, int VEC, int G, int PL>
__global__ void __launch_bounds__(G > 256 ? G : 256) fwd_kernel(const FwdArgs p) {
    constexpr int NT = G > 256 ? G : 256, R = NT / G, AE = ABF ? 2 : 4, SE = SBF ? 2 : 4;
    __shared__ float lds[G > 64 ? 16 : 1];
    const int g = threadIdx.x % G;
    Slice<ABF, VEC, PL> uv, gv;
    Slice<SBF, VEC, PL> xv;
    const long long step = (long long)gridDim.x * R;
    long long mine = (long long)blockIdx.x * R + threadIdx.x / G;
    auto ask = [&](long long row) {                       // (lanes without a row take the last one's, and keep quiet)
        const size_t t = row < p.T ? row : p.T - 1;
        uv.template load<G>(p.u + t * p.us, g, p.C);
        if (p.gate) gv.template load<G>(p.gate + t * p.gs, g, p.C);
        xv.template load<G>(p.residual + t * p.rs, g, p.C);
    };
    ask(mine);
    float pw[PL], pb[PL], sc[PL], qw[PL], qb[PL];
    load_param<VEC, G, PL>(pw, p.par[0], p.w_bf16, g, p.C, 1.f);
    load_param<VEC, G, PL>(pb, p.par[1], p.w_bf16, g, p.C, 0.f);
    load_param<VEC, G, PL>(sc, p.par[2], p.w_bf16, g, p.C, 1.f);
    load_param<VEC, G, PL>(qw, p.par[3], p.w_bf16, g, p.C, 1.f);
    load_param<VEC, G, PL>(qb, p.par[4], p.w_bf16, g, p.C, 0.f);
    for (long long t0 = (long long)blockIdx.x * R; t0 < p.T; t0 += step, mine += step) {
        const bool real = mine < p.T;
        const size_t t = mine;
        float v[PL], x[PL], pm = 0.f, pr = 1.f, qm = 0.f, qr = 1.f;
        uv.to_f32(v);
        if (p.par[0]) {
            statistics<VEC, G, PL>(v, g, p.C, p.rms, p.eps, pm, pr, lds);
#pragma unroll
            for (int j = 0; j < PL; ++j) v[j] = fmaf((v[j] - pm) * pr, pw[j], pb[j]);
        }
        if (p.gate) {
            float ga[PL];
            gv.to_f32(ga);
#pragma unroll
            for (int j = 0; j < PL; ++j) v[j] *= ga[j] * sigmoid_f32(ga[j]);
        }
        xv.to_f32(x);
        if (t0 + step < p.T) ask(mine + step);
#pragma unroll
        for (int j = 0; j < PL; ++j) x[j] = ((j / VEC) * G + g) * VEC < p.C ? fmaf(sc[j], v[j], x[j]) : 0.f;
        Slice<SBF, VEC, PL> ov;
        ov.from_f32(x);
        if (real) ov.template store<G>(p.out + t * p.C * SE, g, p.C);
        if (p.par[3]) {
            statistics<VEC, G, PL>(x, g, p.C, p.rms, p.eps, qm, qr, lds);
            if (p.normed) {
#pragma unroll
                for (int j = 0; j < PL; ++j) x[j] = fmaf((x[j] - qm) * qr, qw[j], qb[j]);
                Slice<ABF, VEC, PL> nv;
                nv.from_f32(x);
                if (real) nv.template store<G>(p.normed + t * p.C * AE, g, p.C);
            }
        }
        if (p.stats && real && g == 0) ((float4*)p.stats)[t] = make_float4(pm, pr, qm, qr);
    }
}

// The forward's out is formed again in fp32 from the same inputs. Bound by memory as the forward is: the calls named there 421 us (5.1 TB/s), 160 us (5.3 TB/s)
// and 34 us, the last of them in loads of a channel each and in joining the blocks' sums (T=50021, C=1001: fp32 325 us, 4.9 TB/s, but bf16, two bytes a load, 517 us,
// 1.6 TB/s). One wave a SIMD as the least: with the compiler's own choice of registers 454 us for the first one where this then took 435.
template <bool ABF, bool SBF, int VEC, int G, int PL>
__global__ void __launch_bounds__(G > 256 ? G : 256, 1) bwd_kernel(const BwdArgs p) {
    constexpr int NT = G > 256 ? G : 256, R = NT / G, AE = ABF ? 2 : 4, SE = SBF ? 2 : 4;
    __shared__ float lds[G > 64 ? 32 : 1];
    __shared__ float part[R > 1 ? R : 1][R > 1 ? G * PL : 1];
    const int g = threadIdx.x % G;
    float pw[PL], pb[PL], sc[PL], qw[PL];
    load_param<VEC, G, PL>(pw, p.par[0], p.w_bf16, g, p.C, 1.f);
    load_param<VEC, G, PL>(pb, p.par[1], p.w_bf16, g, p.C, 0.f);
    load_param<VEC, G, PL>(sc, p.par[2], p.w_bf16, g, p.C, 1.f);
    load_param<VEC, G, PL>(qw, p.par[3], p.w_bf16, g, p.C, 1.f);
    float sum[kParams][PL] = {};
    const float inv = 1.f / p.C;
    for (long long t0 = (long long)blockIdx.x * R; t0 < p.T; t0 += (long long)gridDim.x * R) {
        const long long mine = t0 + threadIdx.x / G;
        const bool real = R == 1 || mine < p.T;
        const size_t t = real ? mine : p.T - 1;
        Slice<ABF, VEC, PL> uv, gv, nv;
        Slice<SBF, VEC, PL> xv, ov;
        const int there = real ? p.C : 0;                 // (lanes without a row have zeros, which add nothing; a 0 times what another row holds may be NaN)
        uv.template load<G>(p.u + t * p.us, g, there);
        if (p.gate) gv.template load<G>(p.gate + t * p.gs, g, there);
        xv.template load<G>(p.residual + t * p.rs, g, there);
        if (p.dout) ov.template load<G>(p.dout + t * p.os, g, there);
        if (p.dnormed) nv.template load<G>(p.dnormed + t * p.ns, g, there);
        float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
        if (real) st = ((const float4*)p.stats)[t];
        const float pm = st.x, pr = st.y, qm = st.z, qr = st.w;
        float n[PL], v[PL], d[PL], ga[PL], x[PL];
        uv.to_f32(n);
        if (p.par[0])
#pragma unroll
            for (int j = 0; j < PL; ++j) n[j] = (n[j] - pm) * pr;
#pragma unroll
        for (int j = 0; j < PL; ++j) v[j] = fmaf(n[j], pw[j], pb[j]), d[j] = 0.f;
        if (p.gate) {
            gv.to_f32(ga);
#pragma unroll
            for (int j = 0; j < PL; ++j) v[j] *= ga[j] * sigmoid_f32(ga[j]);
        }
        if (p.dout) ov.to_f32(d);
        if (p.par[3] && p.dnormed) {
            float dn[PL], s[2] = {0.f, 0.f};
            xv.to_f32(x);
            nv.to_f32(dn);
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                const bool in = ((j / VEC) * G + g) * VEC < p.C;
                x[j] = in ? (fmaf(sc[j], v[j], x[j]) - qm) * qr : 0.f;
                sum[3][j] = fmaf(dn[j], x[j], sum[3][j]);
                sum[4][j] += dn[j];
                dn[j] *= qw[j];
                s[0] += dn[j];
                s[1] = fmaf(dn[j], x[j], s[1]);
            }
            group_sum<G, 2>(s, lds);
            const float m0 = p.rms ? 0.f : s[0] * inv, m1 = s[1] * inv;
#pragma unroll
            for (int j = 0; j < PL; ++j) d[j] = fmaf(qr, dn[j] - m0 - x[j] * m1, d[j]);
        }
        ov.from_f32(d);
        if (real) ov.template store<G>(p.dresidual + t * p.C * SE, g, p.C);
#pragma unroll
        for (int j = 0; j < PL; ++j) {
            sum[2][j] = fmaf(d[j], v[j], sum[2][j]);
            d[j] *= sc[j];
        }
        if (p.gate) {
            float dg[PL];
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                const float sg = sigmoid_f32(ga[j]);
                dg[j] = d[j] * fmaf(n[j], pw[j], pb[j]) * sg * fmaf(ga[j], 1.f - sg, 1.f);
                d[j] *= ga[j] * sg;
            }
            gv.from_f32(dg);
            if (real) gv.template store<G>(p.dgate + t * p.C * AE, g, p.C);
        }
        if (p.par[0]) {
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                sum[0][j] = fmaf(d[j], n[j], sum[0][j]);
                sum[1][j] += d[j];
                d[j] *= pw[j];
                const bool in = ((j / VEC) * G + g) * VEC < p.C;
                s[0] += in ? d[j] : 0.f;
                s[1] = in ? fmaf(d[j], n[j], s[1]) : s[1];
            }
            group_sum<G, 2>(s, lds);
            const float m0 = p.rms ? 0.f : s[0] * inv, m1 = s[1] * inv;
#pragma unroll
            for (int j = 0; j < PL; ++j) d[j] = pr * (d[j] - m0 - n[j] * m1);
        }
        uv.from_f32(d);
        if (real) uv.template store<G>(p.du + t * p.C * AE, g, p.C);
    }
#pragma unroll
    for (int i = 0; i < kParams; ++i) {
        if (!(p.want >> i & 1)) continue;
        float* to = p.partial + ((size_t)blockIdx.x * kParams + i) * p.C;
        if constexpr (R > 1) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PL; ++j) part[threadIdx.x / G][((j / VEC) * G + g) * VEC + j % VEC] = sum[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < p.C; c += NT) {
                float s = 0.f;
#pragma unroll
                for (int r = 0; r < R; ++r) s += part[r][c];
                to[c] = s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < PL; ++j) {
                const int c = ((j / VEC) * G + g) * VEC + j % VEC;
                if (c < p.C) to[c] = sum[i][j];
            }
        }
    }
}

// Adds up the blocks' sums of a parameter's gradient, in fp64: 16 columns a block, each of its 64 groups of lanes every 64th block's sums, eight
// loads at a time, then the groups'.
struct SumArgs {
    const float* partial;
    void* out[kParams];
    int blocks, C, g_bf16;
};
__global__ void __launch_bounds__(1024) sum_kernel(const SumArgs p) {
    __shared__ double part[64][16];
    const int i = blockIdx.y, j = threadIdx.x / 16, lane = threadIdx.x % 16, c = blockIdx.x * 16 + lane;
    if (!p.out[i]) return;
    double s = 0;
    if (c < p.C) {
        const float* at = p.partial + (size_t)i * p.C + c;
        const size_t step = (size_t)kParams * p.C;
        int b = j;
        for (; b + 7 * 64 < p.blocks; b += 8 * 64) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = at[(b + u * 64) * step];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        for (; b < p.blocks; b += 64) s += at[b * step];
    }
    part[j][lane] = s;
    __syncthreads();
    if (j || c >= p.C) return;
    s = 0;
#pragma unroll 8
    for (int w = 0; w < 64; ++w) s += part[w][lane];
    if (p.g_bf16) ((uint16_t*)p.out[i])[c] = f32_to_bf16((float)s);
    else ((float*)p.out[i])[c] = (float)s;
}

}  // namespace rn
}  // namespace nplm
