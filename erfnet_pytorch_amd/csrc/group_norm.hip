// Group normalisation with an activation on channels-last maps [N][HW][C], forward and backward.
//
//     u = (x - mean) rstd gamma_c + beta_c,  y = act(u);  mean, rstd over the HW x C/G values of (image n, group g)
//     du = dy act'(u),  A_nc = sum_hw du,  B_nc = sum_hw du xhat,  dbeta = sum_n A,  dgamma = sum_n B
//     dx = rstd (gamma du - (s1 + xhat s2) / M),  s1 = sum_c gamma A,  s2 = sum_c gamma B over the group,  M = HW C/G
//
// u is formed as (x - mean) (rstd gamma) + beta by one function in both directions, so that the backward pass sees the
// forward pass's signs; folding the mean into a shift instead would cost u its digits where |mean| is far above the spread.
#include "../../include/erfnet_mi355.h"
#include "common.cuh"

__device__ __forceinline__ float gn_u(float x, float mean, float a, float beta) { return fmaf(x - mean, a, beta); }

template <int ACT>
__device__ __forceinline__ float gn_act(float u) {
    if (ACT == ERF_ACT_RELU) return u < 0.f ? 0.f : u;                  // NaN stays
    if (ACT == ERF_ACT_SILU) return u / (1.f + __expf(-u));
    return u;
}
template <int ACT>
__device__ __forceinline__ float gn_slope(float u) {
    if (ACT == ERF_ACT_RELU) return u > 0.f ? 1.f : 0.f;
    if (ACT == ERF_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-u));
        return s * (1.f + u * (1.f - s));
    }
    return 1.f;
}

struct GnArgs {
    const void *x, *dy;
    void *y, *dx;
    const float *gamma, *beta;
    float *mean, *rstd, *dgamma, *dbeta, *sums;       // sums: [N][C][2] of A, B
    long long HW;
    int N, C, G;
    float eps;
};

__device__ __forceinline__ float block_sum(float v, float* sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// One workgroup per (image, group): three passes over the group's values.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void gn_fwd_group_kernel(const GnArgs a) {
    __shared__ float sh[4];
    const int n = blockIdx.x / a.G, g = blockIdx.x % a.G, cpg = a.C / a.G;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.C + g * cpg;
    T* y = (T*)a.y + (long long)n * a.HW * a.C + g * cpg;
    const long long m = a.HW * cpg;
    float s = 0.f;
    for (long long i = threadIdx.x; i < m; i += 256) s += Elem<T>::ld(x + i / cpg * a.C + i % cpg);
    const float mean = block_sum(s, sh) / (float)m;
    s = 0.f;
    for (long long i = threadIdx.x; i < m; i += 256) {
        const float d = Elem<T>::ld(x + i / cpg * a.C + i % cpg) - mean;
        s += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(s, sh) / (float)m + a.eps);
    if (threadIdx.x == 0) { a.mean[blockIdx.x] = mean; a.rstd[blockIdx.x] = rstd; }
    for (long long i = threadIdx.x; i < m; i += 256) {
        const int c = g * cpg + (int)(i % cpg);
        const long long at = i / cpg * a.C + i % cpg;
        const float u = gn_u(Elem<T>::ld(x + at), mean, rstd * (a.gamma ? a.gamma[c] : 1.f), a.beta ? a.beta[c] : 0.f);
        Elem<T>::st(y + at, gn_act<ACT>(u));
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_group_kernel(const GnArgs a) {
    __shared__ float sh[4];
    const int n = blockIdx.x / a.G, g = blockIdx.x % a.G, cpg = a.C / a.G;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.C;
    const T* dy = (const T*)a.dy + (long long)n * a.HW * a.C;
    T* dx = (T*)a.dx + (long long)n * a.HW * a.C;
    const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x], m = (float)(a.HW * cpg);
    float s1 = 0.f, s2 = 0.f;
    for (int c = g * cpg; c < (g + 1) * cpg; ++c) {
        const float gamma = a.gamma ? a.gamma[c] : 1.f, beta = a.beta ? a.beta[c] : 0.f;
        float p = 0.f, q = 0.f;
        for (long long i = threadIdx.x; i < a.HW; i += 256) {
            const float v = Elem<T>::ld(x + i * a.C + c);
            const float du = Elem<T>::ld(dy + i * a.C + c) * gn_slope<ACT>(gn_u(v, mean, rstd * gamma, beta));
            p += du;
            q += du * ((v - mean) * rstd);
        }
        p = block_sum(p, sh);
        q = block_sum(q, sh);
        if (threadIdx.x == 0) { a.sums[2 * ((long long)n * a.C + c)] = p; a.sums[2 * ((long long)n * a.C + c) + 1] = q; }
        s1 += gamma * p;
        s2 += gamma * q;
    }
    s1 /= m;
    s2 /= m;
    for (int c = g * cpg; c < (g + 1) * cpg; ++c) {
        const float gamma = a.gamma ? a.gamma[c] : 1.f, beta = a.beta ? a.beta[c] : 0.f;
        for (long long i = threadIdx.x; i < a.HW; i += 256) {
            const float v = Elem<T>::ld(x + i * a.C + c);
            const float du = Elem<T>::ld(dy + i * a.C + c) * gn_slope<ACT>(gn_u(v, mean, rstd * gamma, beta));
            Elem<T>::st(dx + i * a.C + c, rstd * (gamma * du - s1 - (v - mean) * rstd * s2));
        }
    }
}

// dbeta = sum_n A, dgamma = sum_n B
__global__ void gn_param_grads_kernel(const GnArgs a) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= a.C) return;
    double p = 0, q = 0;
    for (int n = 0; n < a.N; ++n) {
        p += a.sums[2 * ((long long)n * a.C + c)];
        q += a.sums[2 * ((long long)n * a.C + c) + 1];
    }
    if (a.dbeta) a.dbeta[c] = (float)p;
    if (a.dgamma) a.dgamma[c] = (float)q;
}

static inline bool gn_shape_ok(int dtype, int N, long long HW, int C, int groups, int act) {
    return (dtype == ERF_F32 || dtype == ERF_BF16) && N > 0 && HW > 0 && C > 0 && groups > 0 && C % groups == 0 && act >= 0 && act <= 2 &&
           (long long)N * groups <= 0x7FFFFFFFll && HW <= (1ll << 40) / C;
}

#define GN_PICK(KERNEL, GRID)                                                                                               \
    do {                                                                                                                    \
        hipStream_t s = (hipStream_t)stream;                                                                                \
        const dim3 grid(GRID), block(256);                                                                                  \
        if (dtype == ERF_F32) {                                                                                             \
            if (act == ERF_ACT_RELU) hipLaunchKernelGGL((KERNEL<float, ERF_ACT_RELU>), grid, block, 0, s, a);               \
            else if (act == ERF_ACT_SILU) hipLaunchKernelGGL((KERNEL<float, ERF_ACT_SILU>), grid, block, 0, s, a);          \
            else hipLaunchKernelGGL((KERNEL<float, ERF_ACT_NONE>), grid, block, 0, s, a);                                   \
        } else {                                                                                                            \
            if (act == ERF_ACT_RELU) hipLaunchKernelGGL((KERNEL<bf16raw, ERF_ACT_RELU>), grid, block, 0, s, a);             \
            else if (act == ERF_ACT_SILU) hipLaunchKernelGGL((KERNEL<bf16raw, ERF_ACT_SILU>), grid, block, 0, s, a);        \
            else hipLaunchKernelGGL((KERNEL<bf16raw, ERF_ACT_NONE>), grid, block, 0, s, a);                                 \
        }                                                                                                                   \
    } while (0)

extern "C" {

size_t erf_group_norm_workspace_bytes(int dtype, int N, long long HW, int C, int groups) {
    if (!gn_shape_ok(dtype, N, HW, C, groups, 0)) return 0;
    return (size_t)N * C * 2 * sizeof(float);
}

int erf_group_norm_fwd(const void* x, void* y, int dtype, int N, long long HW, int C, int groups, const float* gamma, const float* beta,
                       float eps, int act, float* mean, float* rstd, void* workspace, void* stream) {
    if (!x || !y || !mean || !rstd || !workspace || !(eps >= 0) || !gn_shape_ok(dtype, N, HW, C, groups, act)) return ERF_EINVAL;
    GnArgs a = {};
    a.x = x; a.y = y; a.gamma = gamma; a.beta = beta; a.mean = mean; a.rstd = rstd; a.HW = HW; a.N = N; a.C = C; a.G = groups; a.eps = eps;
    GN_PICK(gn_fwd_group_kernel, (unsigned)(N * groups));
    return erf_check_launch();
}

int erf_group_norm_bwd(const void* x, const void* dy, void* dx, int dtype, int N, long long HW, int C, int groups, const float* gamma,
                       const float* beta, int act, const float* mean, const float* rstd, float* dgamma, float* dbeta, void* workspace,
                       void* stream) {
    if (!x || !dy || !dx || !mean || !rstd || !workspace || !gn_shape_ok(dtype, N, HW, C, groups, act)) return ERF_EINVAL;
    GnArgs a = {};
    a.x = x; a.dy = dy; a.dx = dx; a.gamma = gamma; a.beta = beta; a.mean = (float*)mean; a.rstd = (float*)rstd; a.dgamma = dgamma;
    a.dbeta = dbeta; a.sums = (float*)workspace; a.HW = HW; a.N = N; a.C = C; a.G = groups;
    GN_PICK(gn_bwd_group_kernel, (unsigned)(N * groups));
    if (dgamma || dbeta) hipLaunchKernelGGL(gn_param_grads_kernel, dim3((C + 255) / 256), dim3(256), 0, (hipStream_t)stream, a);
    return erf_check_launch();
}

}  // extern "C"
