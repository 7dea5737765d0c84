// Rows of a norm in registers: G lanes (a power of two, 2 to 1024: part of a wave, a wave or a block of waves) have a row, each PL of its channels in vectors
// of VEC adjacent ones. Of the residual norm and the layer norm.
#pragma once
#include "dwconv_device.h"

namespace nplm {
namespace rn {

// Stores past the caches, where a wave's fill whole cache lines: bf16 forward 277 -> 263 us, backward 440 -> 434 (131072 rows, C=1024, kernels as they were then). Where a store fills
// every other 16 bytes of a line (an fp32 stream in vectors of 8) they cost 3 %.
__device__ __forceinline__ void store_nt(const RowVec<true, 8>& r, char* p) {
    __builtin_nontemporal_store((u32x4){r.d[0], r.d[1], r.d[2], r.d[3]}, (u32x4*)p);
}
__device__ __forceinline__ void store_nt(const RowVec<false, 4>& r, char* p) {
    __builtin_nontemporal_store((f32x4){r.v[0], r.v[1], r.v[2], r.v[3]}, (f32x4*)p);
}

// One lane's PL channels of a row, as stored.
template <bool BF16, int VEC, int PL> struct Slice {
    static constexpr int NV = PL / VEC, E = BF16 ? 2 : 4, W = !BF16 && VEC == 8 ? 4 : VEC, M = VEC / W;
    RowVec<BF16, W> d[NV * M];
    template <int G> __device__ __forceinline__ void load(const char* row, int g, int C) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * G + g) * VEC;
#pragma unroll
            for (int m = 0; m < M; ++m)
                if (c < C) d[j * M + m].load(row + (uint32_t)(c + m * W) * E);
                else { const float z[W] = {}; d[j * M + m].from_f32(z); }
        }
    }
    template <int G> __device__ __forceinline__ void store(char* row, int g, int C) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * G + g) * VEC;
#pragma unroll
            for (int m = 0; m < M; ++m)
                if (c < C) {
                    char* at = row + (uint32_t)(c + m * W) * E;
                    if constexpr (M == 1 && W * E == 16) store_nt(d[j], at); else d[j * M + m].store(at);
                }
        }
    }
    __device__ __forceinline__ void to_f32(float (&f)[PL]) const {
#pragma unroll
        for (int j = 0; j < NV * M; ++j) {
            float t[W];
            d[j].to_f32(t);
#pragma unroll
            for (int i = 0; i < W; ++i) f[j * W + i] = t[i];
        }
    }
    __device__ __forceinline__ void from_f32(const float (&f)[PL]) {
#pragma unroll
        for (int j = 0; j < NV * M; ++j) {
            float t[W];
#pragma unroll
            for (int i = 0; i < W; ++i) t[i] = f[j * W + i];
            d[j].from_f32(t);
        }
    }
};

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
typedef uint32_t u2x __attribute__((ext_vector_type(2)));
// Sum over the G lanes of a group, the same bits in each of them (both sides of every exchange add the same two numbers). N sums at once.
template <int G, int N> __device__ __forceinline__ void group_sum(float (&v)[N], float* lds) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] += dpp<0xB1>(v[i]);       // lanes xor 1, xor 2, the other half of 8, the other half of 16
        if constexpr (G >= 4) v[i] += dpp<0x4E>(v[i]);
        if constexpr (G >= 8) v[i] += dpp<0x141>(v[i]);
        if constexpr (G >= 16) v[i] += dpp<0x140>(v[i]);
        if constexpr (G >= 32) {
            const u2x r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
            v[i] = __uint_as_float(r.x) + __uint_as_float(r.y);
        }
        if constexpr (G >= 64) {
            const u2x r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
            v[i] = __uint_as_float(r.x) + __uint_as_float(r.y);
        }
    }
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) lds[i * 16 + wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) s += lds[i * 16 + wave / W * W + w];
            v[i] = s;
        }
        __syncthreads();
    }
}

// One lane's PL channels of a parameter, in vectors where rows are.
template <int VEC, int G, int PL> __device__ __forceinline__ void load_param(float (&o)[PL], const void* p, int bf16, int g, int C, float none) {
#pragma unroll
    for (int j = 0; j < PL; ++j) o[j] = none;
    if (!p) return;
    if (bf16) {
        Slice<true, VEC, PL> d;
        d.template load<G>((const char*)p, g, C);
        d.to_f32(o);
    } else {
        Slice<false, VEC, PL> d;
        d.template load<G>((const char*)p, g, C);
        d.to_f32(o);
    }
}

// mean and 1 / sqrt(var + eps) of a row, the variance from the differences to the mean
template <int VEC, int G, int PL> __device__ __forceinline__ void statistics(const float (&a)[PL], int g, int C, int rms, float eps, float& mean, float& rstd, float* lds) {
    float s[1] = {0.f};
    mean = 0.f;
    if (!rms) {
#pragma unroll
        for (int j = 0; j < PL; ++j) s[0] += a[j];        // (zero beyond C)
        group_sum<G, 1>(s, lds);
        mean = s[0] / C;
    }
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < PL; ++j) {
        const float d = ((j / VEC) * G + g) * VEC < C ? a[j] - mean : 0.f;
        s[0] = fmaf(d, d, s[0]);
    }
    group_sum<G, 1>(s, lds);
    rstd = 1.f / sqrtf(s[0] / C + eps);
}

}  // namespace rn
}  // namespace nplm
