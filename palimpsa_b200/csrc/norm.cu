// Residual addition and RMS norm, forward and backward (sm_100a):
//     z = x + res      y = z w r,  r = 1 / sqrt(mean(z^2) + eps)
//     dz_total = dz + r (w dy - z r^2 mean(w dy z))      dx = dres = dz_total      dw = sum over rows of dy z r
// HBM-bound: one pass over a row, which stays in registers between its sums and what they are used for.  The backward works r
// out again (its sum is taken beside the one it needs anyway) and keeps dw of its channels in registers over all its rows; the
// CTAs' shares are rows of a workspace, summed in a fixed order by a second kernel.
// 32768 x 768, bfloat16 with a float32 residual: forward 60 us (5.0 TB/s), backward 85 (4.7 TB/s).
#include "norm.cuh"

namespace palimpsa {

namespace {

template <int DT, int RT, int TPR, int NC>
__global__ void __launch_bounds__(norm_threads<TPR>(), norm_ctas_per_sm<TPR, NC>()) norm_fwd_kernel(const NormArgs g) {
    constexpr int RPC = norm_threads<TPR>() / TPR;
    __shared__ float scratch[TPR / 32][1];
    const palimpsa_rms_norm& a = g.a;
    const Chunks<NC> ch(threadIdx.x % TPR, TPR, a.D);
    float w[NC][8];
    ld_weight<NC>(a.weight, ch, w);
    const long long step = (long long)gridDim.x * RPC;
    long long row = (long long)blockIdx.x * RPC + threadIdx.x / TPR;
    RowZ<DT, RT, NC> next;
    if (row < a.rows) next.ask(a, row, ch, g.vec);
    for (; row < a.rows; row += step) {
        float z[NC][8], ss[1] = {0.f};
        const RowZ<DT, RT, NC> now = next;
        if (row + step < a.rows) next.ask(a, row + step, ch, g.vec);
        now.take(a, row, ch, g.vec, z);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[0] = fmaf(z[i][e], z[i][e], ss[0]);
        row_add<TPR>(ss, scratch);
        const float r = __frsqrt_rn(ss[0] / (float)a.D + (float)a.eps);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) z[i][e] *= r * w[i][e];
            if (ch.live[i] > 0) st_n<DT, 8>(a.y, row * a.D + ch.c[i], ch.live[i], g.vec, z[i]);
        }
    }
}

template <int DT, int RT, int TPR, int NC>
__global__ void __launch_bounds__(norm_threads<TPR>(), norm_ctas_per_sm<TPR, NC>()) norm_bwd_kernel(const NormArgs g) {
    constexpr int RPC = norm_threads<TPR>() / TPR, ST = RT == NO_RES ? DT : RT;
    __shared__ float scratch[TPR / 32][2];
    __shared__ float sums[RPC > 1 ? RPC : 1][RPC > 1 ? TPR * NC * 8 : 1];
    const palimpsa_rms_norm& a = g.a;
    const Chunks<NC> ch(threadIdx.x % TPR, TPR, a.D);
    float w[NC][8], dw[NC][8];
    ld_weight<NC>(a.weight, ch, w);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
    const void* zp = RT == NO_RES ? a.x : a.z;
    const long long zs = RT == NO_RES ? a.x_stride : a.D;
    const long long step = (long long)gridDim.x * RPC;
    long long row = (long long)blockIdx.x * RPC + threadIdx.x / TPR;
    RowPart<ST, NC> nz, nr;
    RowPart<DT, NC> nd;
    auto ask = [&](long long r) __attribute__((always_inline)) {
        nz.ask(zp, r * zs, ch, g.vec);
        nd.ask(a.dy, r * a.D, ch, g.vec);
        if (a.dz) nr.ask(a.dz, r * a.D, ch, g.vec);
    };
    if (row < a.rows) ask(row);
    for (; row < a.rows; row += step) {
        float z[NC][8], dy[NC][8], dz[NC][8], s[2] = {0.f, 0.f};
        nz.take(zp, row * zs, ch, g.vec, z);
        nd.take(a.dy, row * a.D, ch, g.vec, dy);
        if (a.dz) {
            nr.take(a.dz, row * a.D, ch, g.vec, dz);
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) dz[i][e] = 0.f;
        }
        if (row + step < a.rows) ask(row + step);
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[0] = fmaf(z[i][e], z[i][e], s[0]);
                s[1] = fmaf(w[i][e] * dy[i][e], z[i][e], s[1]);
            }
        row_add<TPR>(s, scratch);
        const float r = __frsqrt_rn(s[0] / (float)a.D + (float)a.eps), k = r * r * (s[1] / (float)a.D);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[i][e] = fmaf(dy[i][e], z[i][e] * r, dw[i][e]);
                dz[i][e] += r * (w[i][e] * dy[i][e] - z[i][e] * k);
            }
            if (ch.live[i] > 0) {
                st_n<DT, 8>(a.dx, row * a.D + ch.c[i], ch.live[i], g.vec, dz[i]);
                if (a.dres) st_n<ST, 8>(a.dres, row * a.D + ch.c[i], ch.live[i], g.vec, dz[i]);
            }
        }
    }
    float* part = reinterpret_cast<float*>(a.workspace) + (long long)blockIdx.x * a.D;
    if constexpr (RPC > 1) {
        const int t = threadIdx.x % TPR, rg = threadIdx.x / TPR;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[rg][(t + i * TPR) * 8 + e] = dw[i][e];
        __syncthreads();
        for (int c = threadIdx.x; c < a.D; c += norm_threads<TPR>()) {
            float x = sums[0][c];
#pragma unroll
            for (int k = 1; k < RPC; ++k) x += sums[k][c];
            part[c] = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < ch.live[i]) part[ch.c[i] + e] = dw[i][e];
    }
}

__global__ void __launch_bounds__(256) norm_finish_kernel(const float* part, int parts, long long D, float* dweight) {
    __shared__ float s[16][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const long long c = (long long)blockIdx.x * 16 + x;
    float acc = 0.f;
    if (c < D)
        for (int p = y; p < parts; p += 16) acc += part[p * D + c];
    s[y][x] = acc;
    __syncthreads();
    if (y == 0 && c < D) {
#pragma unroll
        for (int k = 1; k < 16; ++k) acc += s[k][x];
        dweight[c] = acc;
    }
}

int launched() { return cudaGetLastError() == cudaSuccess ? PALIMPSA_OK : PALIMPSA_E_LAUNCH; }

// CTAs of the backward, by the width of the rows alone: each one's sums are a row of the workspace.
long long bwd_parts(const palimpsa_rms_norm& a) {
    if (a.D <= 256) return norm_ctas<32, 1>(a);
    if (a.D <= 512) return norm_ctas<32, 2>(a);
    if (a.D <= 1024) return norm_ctas<128, 1>(a);
    if (a.D <= 2048) return norm_ctas<128, 2>(a);
    if (a.D <= 4096) return norm_ctas<256, 2>(a);
    if (a.D <= 8192) return norm_ctas<512, 2>(a);
    return norm_ctas<512, 4>(a);
}

}  // namespace

extern "C" {

size_t palimpsa_rms_norm_workspace_bytes(const palimpsa_rms_norm* a) {
    if (!a || a->D <= 0 || a->rows < 0 || a->D > 16384) return 0;
    return (size_t)(bwd_parts(*a) * a->D) * 4 + 256;
}

int palimpsa_rms_norm_fwd(const palimpsa_rms_norm* a, void* stream) {
    if (int rc = norm_check(a)) return rc;
    if (a->rows == 0) return PALIMPSA_OK;
    if (!a->x || !a->y || (a->res_dtype != NO_RES && (!a->res || !a->z))) return PALIMPSA_E_NULL;
    if (a->out_type != PALIMPSA_NORM_IO && !a->scale) return PALIMPSA_E_NULL;
    bool vec = a->D % 8 == 0 && rows_vec(a->x, a->x_stride, 8, a->io_dtype);
    if (a->res_dtype != NO_RES) vec = vec && rows_vec(a->res, a->D, 8, a->res_dtype) && rows_vec(a->z, a->D, 8, a->res_dtype);
    if (a->out_type == PALIMPSA_NORM_IO) vec = vec && rows_vec(a->y, a->D, 8, a->io_dtype);
    else vec = vec && (reinterpret_cast<uintptr_t>(a->y) & 7) == 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->out_type != PALIMPSA_NORM_IO) return launch_norm_quant(*a, vec, st);
    const NormArgs g{*a, vec};
    return norm_dispatch(*a, [&](auto dt, auto rt, auto tpr, auto nc) {
        constexpr int T = norm_threads<tpr.value>();
        norm_fwd_kernel<dt.value, rt.value, tpr.value, nc.value><<<(unsigned)norm_ctas<tpr.value, nc.value>(*a), T, 0, st>>>(g);
        return launched();
    });
}

int palimpsa_rms_norm_bwd(const palimpsa_rms_norm* a, void* stream) {
    if (int rc = norm_check(a)) return rc;
    if (!a->dweight) return PALIMPSA_E_NULL;
    if (a->rows > 0) {
        if (!(a->res_dtype == NO_RES ? a->x : a->z) || !a->dy || !a->dx) return PALIMPSA_E_NULL;
        if (a->res_dtype != NO_RES && a->res_dtype != a->io_dtype && !a->dres) return PALIMPSA_E_NULL;
    }
    if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255) ||
        a->workspace_bytes < palimpsa_rms_norm_workspace_bytes(a))
        return PALIMPSA_E_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long parts = bwd_parts(*a);
    const int zt = a->res_dtype == NO_RES ? a->io_dtype : a->res_dtype;
    bool vec = a->D % 8 == 0 && rows_vec(a->dy, a->D, 8, a->io_dtype) && rows_vec(a->dx, a->D, 8, a->io_dtype);
    vec = vec && (a->res_dtype == NO_RES ? rows_vec(a->x, a->x_stride, 8, zt) : rows_vec(a->z, a->D, 8, zt));
    if (a->dz) vec = vec && rows_vec(a->dz, a->D, 8, zt);
    if (a->dres) vec = vec && rows_vec(a->dres, a->D, 8, zt);
    const NormArgs g{*a, vec};
    if (parts > 0) {
        const int rc = norm_dispatch(*a, [&](auto dt, auto rt, auto tpr, auto nc) {
            norm_bwd_kernel<dt.value, rt.value, tpr.value, nc.value><<<(unsigned)parts, norm_threads<tpr.value>(), 0, st>>>(g);
            return launched();
        });
        if (rc) return rc;
    }
    norm_finish_kernel<<<(unsigned)((a->D + 15) / 16), 256, 0, st>>>(static_cast<const float*>(a->workspace), (int)parts, a->D, a->dweight);
    return launched();
}

}  // extern "C"

}  // namespace palimpsa
