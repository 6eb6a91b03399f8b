// Shared by the operators of the block around the recurrence (conv.cu, norm.cu, ssm*.cu).
#pragma once

#include "common.cuh"

namespace palimpsa {

__device__ __forceinline__ float warp_add(float x) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
}
__device__ __forceinline__ double warp_add(double x) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
}

// A sequence's token rows.  Offsets come from the device and are clamped, so that wrong ones are never a wild access.
struct Span {
    int n;               // sequence, -1: rows that belong to none
    long long bos, eos;  // its rows
};
__device__ __forceinline__ long long clamped_offset(const int* cu, int i, long long total) {
    const long long x = cu[i];
    return x < 0 ? 0 : (x > total ? total : x);
}
// The span that row t lies in (eos > t always), by a whole warp.
__device__ __forceinline__ Span find_span(const int* cu, int num_seqs, long long seq_len, long long total, long long t, int lane) {
    Span s;
    if (!cu) {
        s.n = (int)(t / seq_len);
        s.bos = s.n * seq_len, s.eos = s.bos + seq_len;
        return s;
    }
    int lo = 0, hi = num_seqs;  // the last n with cu[n] <= t: 32 candidates a step
    if (num_seqs == 0 || clamped_offset(cu, 0, total) > t) {
        s.n = -1, s.bos = 0, s.eos = num_seqs ? clamped_offset(cu, 0, total) : total;
        return s;
    }
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, i < hi && clamped_offset(cu, i < hi ? i : lo, total) <= t);
        const int last = 31 - __clz(m | 1u);
        lo += last * step;
        hi = min(hi, lo + step);
    }
    s.n = lo, s.bos = clamped_offset(cu, lo, total), s.eos = clamped_offset(cu, lo + 1, total);
    if (s.eos <= t) {  // behind the last sequence
        s.n = -1, s.bos = s.eos, s.eos = total;
    }
    return s;
}
__device__ __forceinline__ void seq_span(const int* cu, long long seq_len, long long total, int n, long long& bos, long long& eos) {
    if (!cu) {
        bos = n * seq_len, eos = bos + seq_len;
    } else {
        bos = clamped_offset(cu, n, total), eos = clamped_offset(cu, n + 1, total);
        if (eos < bos) eos = bos;
    }
}

// N = 4 or 8 consecutive values of an io type: in wide accesses where `vec` says that the address allows it.
template <int DT, int N>
__device__ __forceinline__ void ld_n(const void* base, long long idx, int live, bool vec, float (&x)[N]) {
    if (vec) {
        if constexpr (DT == PALIMPSA_F32) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const float4 y = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + idx)[i];
                x[4 * i] = y.x, x[4 * i + 1] = y.y, x[4 * i + 2] = y.z, x[4 * i + 3] = y.w;
            }
        } else {
            unsigned r[N / 2];
            const unsigned short* p = reinterpret_cast<const unsigned short*>(base) + idx;
            if constexpr (N == 8) {
                const uint4 u = *reinterpret_cast<const uint4*>(p);
                r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(p);
                r[0] = u.x, r[1] = u.y;
            }
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                float2 f;
                if (DT == PALIMPSA_BF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r[i]));
                else f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < live ? ld1<DT>(base, idx + i) : 0.f;
    }
}
template <int DT, int N>
__device__ __forceinline__ void st_n(void* base, long long idx, int live, bool vec, const float (&x)[N]) {
    if (vec) {
        if constexpr (DT == PALIMPSA_F32) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i)
                reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + idx)[i] =
                    make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
            unsigned r[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                if (DT == PALIMPSA_BF16) {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                    r[i] = *reinterpret_cast<const unsigned*>(&h);
                } else {
                    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                    r[i] = *reinterpret_cast<const unsigned*>(&h);
                }
            }
            unsigned short* p = reinterpret_cast<unsigned short*>(base) + idx;
            if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
            else *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < live) st1(base, idx + i, x[i], DT);
    }
}

// Host: may rows of `stride` elements at p be read N elements at a time?
inline bool rows_vec(const void* p, long long stride, int n, int dtype) {
    const size_t bytes = (size_t)n * dtype_size(dtype);
    return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && stride % n == 0;
}

}  // namespace palimpsa
