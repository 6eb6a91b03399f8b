// Residual addition and RMS norm with an output in 8 bits and its scales (sm_100a):
//     y = z w r      s = max(amax |y|, 2^-100) / top, rounded to float32      q = y / s to the nearest 8-bit value, ties to even
// with one s per row, or per row and `block` channels.  HBM-bound, one pass over a row.
//
// The 8-bit values are those of 64-bit arithmetic, so that they do not depend on the order of a sum: sum z^2 is taken in 64 bits
// (exact products), z w is held as a rounded product and its remainder, the largest of a row or block is found by both, and r and
// s are worked out in 64 bits.  An element then takes one multiplication in float32, y/s = (z w)(r/s) with a relative error
// below 3 * 2^-24; only where that is within 8 steps of float32 of the middle between two 8-bit values (one element in 2^15) it
// is worked out in 64 bits too.
#include <cuda_fp8.h>

#include "norm.cuh"

namespace palimpsa {

namespace {

// The float32 that rounds to the same 8-bit value as t: towards zero, with the last bit set where that was not exact.
__device__ __forceinline__ float to_odd(double t) {
    const float f = __double2float_rz(t);
    return (double)f == t ? f : __uint_as_float(__float_as_uint(f) | 1u);
}
// Is t too near the middle of two neighbouring values for its error?
template <int OUT>
__device__ __forceinline__ bool in_doubt(float t) {
    const float m = fabsf(t);
    if (OUT == PALIMPSA_NORM_E4M3) {  // 3 bits of mantissa are kept; below 2^-6 the step is 2^-9, as between 2^-6 and 2^-5
        const unsigned u = __float_as_uint(m < 0x1p-6f ? m + 0x1p-6f : m) & 0xfffffu;
        return u - 0x7fff8u <= 16u;
    }
    return fabsf(m - floorf(m) - 0.5f) < 0x1p-14f;  // |t| <= 127: an error of 2^-15.4
}
template <int OUT>
__device__ __forceinline__ unsigned eight_bits(float t) {
    if (OUT == PALIMPSA_NORM_E4M3) return (unsigned)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
    const int q = __float2int_rn(t);
    return (unsigned)(q > 127 ? 127 : q < -127 ? -127 : q) & 0xffu;
}
template <int OUT>
__device__ __forceinline__ unsigned pair_bits(float t, float u) {
    if (OUT == PALIMPSA_NORM_E4M3) return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(t, u), __NV_SATFINITE, __NV_E4M3);
    return eight_bits<OUT>(t) | eight_bits<OUT>(u) << 8;
}

// 1 / sqrt(x) and 1 / s in 64 bits, to a few of their last bits: two steps of Newton's method from the float32 value (2^-22, then
// 2^-43, then 2^-53), where that is in range.  The library's square root and division take ten times as many instructions, for
// 8 to 32 elements a thread.
__device__ __forceinline__ double rsqrt64(double x) {
    if (!(x > 1e-30 && x < 1e30)) return 1. / sqrt(x);
    double r = rsqrtf((float)x);
    r = r * fma(-0.5 * x * r, r, 1.5);
    return r * fma(-0.5 * x * r, r, 1.5);
}
__device__ __forceinline__ double rcp64(float s) {
    if (!(s > 1e-35f && s < 1e30f)) return 1. / (double)s;
    double r = __frcp_rn(s);
    r = fma(r, fma(-(double)s, r, 1.), r);
    return fma(r, fma(-(double)s, r, 1.), r);
}

struct Top {  // a value and its remainder, m + l exactly; the largest by m, then by l
    float m, l;
    __device__ __forceinline__ void take(float m2, float l2) {
        if (m2 > m || (m2 == m && l2 > l)) m = m2, l = l2;
    }
};

template <int DT, int RT, int TPR, int NC, int OUT>
__global__ void __launch_bounds__(norm_threads<TPR>()) norm_quant_kernel(const NormArgs g) {
    constexpr int RPC = norm_threads<TPR>() / TPR;
    constexpr double TOP = OUT == PALIMPSA_NORM_E4M3 ? 448. : 127.;
    __shared__ double scratch[TPR / 32][1];
    __shared__ Top tops[TPR / 32];
    const palimpsa_rms_norm& a = g.a;
    const Chunks<NC> ch(threadIdx.x % TPR, TPR, a.D);
    const int blocks = a.block ? (int)((a.D + a.block - 1) / a.block) : 1;
    const double per_channel = 1. / (double)a.D;
    float w[NC][8];
    ld_weight<NC>(a.weight, ch, w);
    for (long long row = (long long)blockIdx.x * RPC + threadIdx.x / TPR; row < a.rows; row += (long long)gridDim.x * RPC) {
        float z[NC][8];
        double ss[1] = {0.};
        ld_z<DT, RT, NC>(a, g.vec, row, ch, z);
        Top top[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            top[i].m = top[i].l = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double d = z[i][e];
                ss[0] = fma(d, d, ss[0]);
                const float hi = z[i][e] * w[i][e], lo = fmaf(z[i][e], w[i][e], -hi);
                top[i].take(fabsf(hi), hi < 0.f ? -lo : lo);
            }
        }
        row_add<TPR>(ss, scratch);
        const double r = rsqrt64(fma(ss[0], per_channel, a.eps));
        // the group that shares a scale: block/8 neighbouring lanes, or the row
        const int lanes = a.block ? a.block / 8 : 32;
        if (!a.block) {
#pragma unroll
            for (int i = 1; i < NC; ++i) top[0].take(top[i].m, top[i].l);
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i > 0 && !a.block) break;
            for (int off = lanes / 2; off >= 1; off >>= 1)
                top[i].take(__shfl_xor_sync(0xffffffffu, top[i].m, off), __shfl_xor_sync(0xffffffffu, top[i].l, off));
        }
        if constexpr (TPR > 32) {
            if (!a.block) {  // the barriers of the next row's sum keep it apart from this one
                if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top[0];
                __syncthreads();
#pragma unroll
                for (int k = 0; k < TPR / 32; ++k) top[0].take(tops[k].m, tops[k].l);
            }
        }
        double factor = 0.;
        float factor32 = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (i == 0 || a.block) {
                const double largest = ((double)top[i].m + (double)top[i].l) * r;
                const float s = (float)((largest < 0x1p-100 ? 0x1p-100 : largest) * (1. / TOP));
                factor = r * rcp64(s);
                factor32 = (float)factor;
                if (a.block) {
                    if (ch.live[i] > 0 && (threadIdx.x & (lanes - 1)) == 0) a.scale[row * blocks + ch.c[i] / a.block] = s;
                } else if (threadIdx.x % TPR == 0) {
                    a.scale[row] = s;
                }
            }
            float t[8];
            bool doubt = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[e] = z[i][e] * w[i][e] * factor32;
                doubt |= in_doubt<OUT>(t[e]);
            }
            if (doubt) {
#pragma unroll 1
                for (int e = 0; e < 8; ++e) {
                    float x = 0.f, y = 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k == e) x = z[i][k], y = w[i][k];
                    const float odd = to_odd((double)x * (double)y * factor);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k == e) t[k] = odd;
                }
            }
            unsigned q[2];
            q[0] = pair_bits<OUT>(t[0], t[1]) | pair_bits<OUT>(t[2], t[3]) << 16;
            q[1] = pair_bits<OUT>(t[4], t[5]) | pair_bits<OUT>(t[6], t[7]) << 16;
            if (ch.live[i] > 0) {
                unsigned char* y = static_cast<unsigned char*>(a.y) + row * a.D + ch.c[i];
                if (g.vec) {
                    *reinterpret_cast<uint2*>(y) = make_uint2(q[0], q[1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (e < ch.live[i]) y[e] = (unsigned char)(q[e / 4] >> (8 * (e % 4)));
                }
            }
        }
    }
}

}  // namespace

int launch_norm_quant(const palimpsa_rms_norm& a, bool vec, cudaStream_t stream) {
    const NormArgs g{a, vec};
    return norm_dispatch(a, [&](auto dt, auto rt, auto tpr, auto nc) {
        constexpr int T = norm_threads<tpr.value>();
        const unsigned ctas = (unsigned)norm_ctas(a, 2048 / T);
        if (a.out_type == PALIMPSA_NORM_E4M3)
            norm_quant_kernel<dt.value, rt.value, tpr.value, nc.value, PALIMPSA_NORM_E4M3><<<ctas, T, 0, stream>>>(g);
        else
            norm_quant_kernel<dt.value, rt.value, tpr.value, nc.value, PALIMPSA_NORM_INT8><<<ctas, T, 0, stream>>>(g);
        return cudaGetLastError() == cudaSuccess ? PALIMPSA_OK : PALIMPSA_E_LAUNCH;
    });
}

}  // namespace palimpsa
