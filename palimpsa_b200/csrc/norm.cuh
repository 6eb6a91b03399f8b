// Residual addition and RMS norm: what norm.cu (output in the io type, backward) and norm_quant.cu (8-bit output) share.
//
// A row is held by TPR threads (a warp up to 512 channels, else a CTA), each with NC chunks of 8 neighbouring channels in
// registers, so that it is read once whatever is done with it.  A CTA takes row after row and keeps its channels' weights.
#pragma once

#include "block.cuh"
#include "host.h"

namespace palimpsa {

// The residual stream's type, RT: NO_RES, the io type, or float32.
constexpr int NO_RES = -1;

template <int TPR>
__host__ __device__ constexpr int norm_threads() { return TPR < 128 ? 128 : TPR; }

struct NormArgs {
    palimpsa_rms_norm a;
    bool vec;  // every row of every tensor may be accessed 8 channels at a time
};

template <int DT>
__device__ __forceinline__ float rounded(float x) {
    if (DT == PALIMPSA_BF16) return __bfloat162float(__float2bfloat16_rn(x));
    if (DT == PALIMPSA_F16) return __half2float(__float2half_rn(x));
    return x;
}

// Sum over the threads of a row, the same bits in each.
template <int TPR, class T, int N>
__device__ __forceinline__ void row_add(T (&x)[N], T (*scratch)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = warp_add(x[i]);
    if constexpr (TPR > 32) {
        __syncthreads();  // the scratch of the row before has been read
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) scratch[threadIdx.x >> 5][i] = x[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = scratch[0][i];
#pragma unroll
            for (int w = 1; w < TPR / 32; ++w) x[i] += scratch[w][i];
        }
    }
}

template <int NC>
struct Chunks {
    long long c[NC];  // first channel
    int live[NC];     // channels, <= 0: none
    __device__ __forceinline__ Chunks(int t, int tpr, long long D) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            c[i] = 8ll * (t + i * tpr);
            const long long left = D - c[i];
            live[i] = left < 0 ? 0 : left > 8 ? 8 : (int)left;
        }
    }
};

// z of a row: loads of all chunks first, then the sums.
template <int DT, int RT, int NC>
__device__ __forceinline__ void ld_z(const palimpsa_rms_norm& a, bool vec, long long row, const Chunks<NC>& ch, float (&z)[NC][8]) {
    constexpr int ST = RT == NO_RES ? DT : RT;
    float r[RT == NO_RES ? 1 : NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        if (ch.live[i] > 0) {
            ld_n<DT, 8>(a.x, row * a.x_stride + ch.c[i], ch.live[i], vec, z[i]);
            if constexpr (RT != NO_RES) ld_n<ST, 8>(a.res, row * a.D + ch.c[i], ch.live[i], vec, r[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] = r[RT == NO_RES ? 0 : i][e] = 0.f;
        }
    }
    if constexpr (RT != NO_RES) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] = rounded<ST>(z[i][e] + r[i][e]);
            if (ch.live[i] > 0) st_n<ST, 8>(a.z, row * a.D + ch.c[i], ch.live[i], vec, z[i]);
        }
    }
}
template <int NC>
__device__ __forceinline__ void ld_weight(const float* weight, const Chunks<NC>& ch, float (&w)[NC][8]) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[i][e] = e < ch.live[i] ? weight[ch.c[i] + e] : 0.f;
}

// f(type of io, type of the residual, threads of a row, chunks of a thread) for a call's types and width.
template <class F>
int norm_dispatch(const palimpsa_rms_norm& a, F&& f) {
    auto width = [&](auto dt, auto rt) {
        using std::integral_constant;
        if (a.D <= 256) return f(dt, rt, integral_constant<int, 32>(), integral_constant<int, 1>());
        if (a.D <= 512) return f(dt, rt, integral_constant<int, 32>(), integral_constant<int, 2>());
        if (a.D <= 1024) return f(dt, rt, integral_constant<int, 128>(), integral_constant<int, 1>());
        if (a.D <= 2048) return f(dt, rt, integral_constant<int, 256>(), integral_constant<int, 1>());
        if (a.D <= 4096) return f(dt, rt, integral_constant<int, 256>(), integral_constant<int, 2>());
        if (a.D <= 8192) return f(dt, rt, integral_constant<int, 512>(), integral_constant<int, 2>());
        return f(dt, rt, integral_constant<int, 512>(), integral_constant<int, 4>());
    };
    using F32 = std::integral_constant<int, PALIMPSA_F32>;
    auto res = [&](auto dt) {
        if (a.res_dtype == NO_RES) return width(dt, std::integral_constant<int, NO_RES>());
        if constexpr (dt.value != PALIMPSA_F32)
            if (a.res_dtype == PALIMPSA_F32) return width(dt, F32());
        return width(dt, dt);
    };
    return a.io_dtype == PALIMPSA_F32 ? res(F32())
           : a.io_dtype == PALIMPSA_BF16 ? res(std::integral_constant<int, PALIMPSA_BF16>())
                                         : res(std::integral_constant<int, PALIMPSA_F16>());
}
inline int norm_row_threads(long long D) { return D <= 512 ? 32 : D <= 1024 ? 128 : D <= 4096 ? 256 : 512; }
inline int norm_check(const palimpsa_rms_norm* a) {
    if (!a) return PALIMPSA_E_NULL;
    if (a->struct_size != sizeof(palimpsa_rms_norm)) return PALIMPSA_E_VERSION;
    if (a->rows < 0 || a->D <= 0 || a->rows > (1ll << 40) || a->x_stride < a->D) return PALIMPSA_E_SHAPE;
    if (a->D > 16384) return PALIMPSA_E_DIM;
    if (a->io_dtype != PALIMPSA_F32 && a->io_dtype != PALIMPSA_BF16 && a->io_dtype != PALIMPSA_F16) return PALIMPSA_E_DTYPE;
    if (a->res_dtype != NO_RES && a->res_dtype != PALIMPSA_F32 && a->res_dtype != a->io_dtype) return PALIMPSA_E_DTYPE;
    if (a->out_type < PALIMPSA_NORM_IO || a->out_type > PALIMPSA_NORM_INT8) return PALIMPSA_E_DTYPE;
    if (a->block != 0 && a->block != 32 && a->block != 64 && a->block != 128 && a->block != 256) return PALIMPSA_E_SHAPE;
    if (!a->weight) return PALIMPSA_E_NULL;
    return PALIMPSA_OK;
}
// CTAs that walk the rows: as many as are resident at once, each row's threads (128 at least) in one.
inline long long norm_ctas(const palimpsa_rms_norm& a, int per_sm) {
    const int tpr = norm_row_threads(a.D), rows_per = tpr < 128 ? 128 / tpr : 1;
    const long long all = (a.rows + rows_per - 1) / rows_per, most = (long long)B200_SMS * per_sm;
    return all < most ? all : most;
}

int launch_norm_quant(const palimpsa_rms_norm& a, bool vec, cudaStream_t stream);

}  // namespace palimpsa
