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

// 8 channels as they lie in memory: what waits in registers while the row before is worked on.
template <int DT>
struct Raw8 {
    uint4 u[DT == PALIMPSA_F32 ? 2 : 1];
    __device__ __forceinline__ void ld(const void* base, long long idx) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + idx * (DT == PALIMPSA_F32 ? 4 : 2));
        u[0] = p[0];
        if constexpr (DT == PALIMPSA_F32) u[1] = p[1];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        if constexpr (DT == PALIMPSA_F32) {
            const unsigned r[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r[i]);
        } else {
            const unsigned r[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 f;
                if (DT == PALIMPSA_BF16) f = make_float2(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
                else f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            }
        }
    }
};
// One tensor's part of a row: asked for ahead where it can be (vec), else when it is taken.
template <int DT, int NC>
struct RowPart {
    Raw8<DT> raw[NC];
    __device__ __forceinline__ void ask(const void* base, long long at, const Chunks<NC>& ch, bool vec) {
        if (!vec) return;
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (ch.live[i] > 0) raw[i].ld(base, at + ch.c[i]);
    }
    __device__ __forceinline__ void take(const void* base, long long at, const Chunks<NC>& ch, bool vec, float (&x)[NC][8]) const {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (ch.live[i] <= 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
            } else if (vec) {
                raw[i].get(x[i]);
            } else {
                ld_n<DT, 8>(base, at + ch.c[i], ch.live[i], false, x[i]);
            }
        }
    }
};
// z of a row: x, or the sum with the residual as it is stored.
template <int DT, int RT, int NC>
struct RowZ {
    static constexpr int ST = RT == NO_RES ? DT : RT;
    RowPart<DT, NC> x;
    RowPart<ST, RT == NO_RES ? 1 : NC> r;
    __device__ __forceinline__ void ask(const palimpsa_rms_norm& a, long long row, const Chunks<NC>& ch, bool vec) {
        x.ask(a.x, row * a.x_stride, ch, vec);
        if constexpr (RT != NO_RES) r.ask(a.res, row * a.D, ch, vec);
    }
    __device__ __forceinline__ void take(const palimpsa_rms_norm& a, long long row, const Chunks<NC>& ch, bool vec, float (&z)[NC][8]) const {
        x.take(a.x, row * a.x_stride, ch, vec, z);
        if constexpr (RT != NO_RES) {
            float y[NC][8];
            r.take(a.res, row * a.D, ch, vec, y);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e) z[i][e] = rounded<ST>(z[i][e] + y[i][e]);
                if (ch.live[i] > 0) st_n<ST, 8>(a.z, row * a.D + ch.c[i], ch.live[i], vec, z[i]);
            }
        }
    }
};
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
        if (a.D <= 2048) return f(dt, rt, integral_constant<int, 128>(), integral_constant<int, 2>());
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
// Threads of an SM that the kernels are compiled for, and CTAs that walk the rows: as many as are resident at once, so that all
// begin together and end together (the backward with 1.14 times as many, and no row ahead: 110 us instead of 85).
template <int TPR, int NC>
__host__ __device__ constexpr int norm_resident() { return NC == 1 ? 768 : 512; }
template <int TPR, int NC>
__host__ __device__ constexpr int norm_ctas_per_sm() {
    return norm_resident<TPR, NC>() / norm_threads<TPR>() < 1 ? 1 : norm_resident<TPR, NC>() / norm_threads<TPR>();
}
template <int TPR, int NC>
long long norm_ctas(const palimpsa_rms_norm& a) {
    constexpr int rows_per = norm_threads<TPR>() / TPR;
    const long long all = (a.rows + rows_per - 1) / rows_per, most = (long long)B200_SMS * norm_ctas_per_sm<TPR, NC>();
    return all < most ? all : most;
}

int launch_norm_quant(const palimpsa_rms_norm& a, bool vec, cudaStream_t stream);

}  // namespace palimpsa
