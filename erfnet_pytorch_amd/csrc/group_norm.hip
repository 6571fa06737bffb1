// Group normalisation with an activation on channels-last maps [N][HW][C], forward and backward.
//
//     u = (x - mean) rstd gamma_c + beta_c,  y = act(u);  mean, rstd over the HW x C/G values of (image n, group g)
//     du = dy act'(u),  A_nc = sum_hw du,  B_nc = sum_hw du xhat,  dbeta = sum_n A,  dgamma = sum_n B
//     dx = rstd (gamma du - (s1 + xhat s2) / M),  s1 = sum_c gamma A,  s2 = sum_c gamma B over the group,  M = HW C/G
//
// u is formed as (x - mean) (rstd gamma) + beta by one function in both directions, so that the backward pass sees the
// forward pass's signs; folding the mean into a shift instead would cost u its digits where |mean| is far above the spread.
//
// By runs of pixels the memory bounds it: x is read twice and y written forward, x and dy are read twice and dx written backward.
// 8 x 524288 x 16 bf16 (134 MB a map), silu: statistics 39 us (3.5 TB/s: one stream and a reduction), apply 48 us (5.6 TB/s), backward
// sums 58 us (4.7 TB/s), apply 70 us (5.7 TB/s).  One pass over the map for both would need every workgroup to wait for all others.  512
// to 4096 workgroups, runs worked off in reverse (what was read last is in the cache) and images one after another changed nothing or
// cost more.  Small maps are bound by the launches: a group per team takes one.
#include "../../include/erfnet_mi355.h"
#include "common.cuh"
#include <type_traits>

template <int N> using Int = std::integral_constant<int, N>;

__device__ __forceinline__ float gn_u(float x, float mean, float a, float beta) { return fmaf(x - mean, a, beta); }

template <int ACT>
__device__ __forceinline__ float gn_act(float u) {
    if (ACT == ERF_ACT_RELU) return u < 0.f ? 0.f : u;                  // NaN stays
    if (ACT == ERF_ACT_SILU) return u * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
    return u;
}
template <int ACT>
__device__ __forceinline__ float gn_slope(float u) {
    if (ACT == ERF_ACT_RELU) return u > 0.f ? 1.f : 0.f;
    if (ACT == ERF_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
        return s * fmaf(u, 1.f - s, 1.f);
    }
    return 1.f;
}

struct GnArgs {
    const void *x, *dy;
    void *y, *dx;
    const float *gamma, *beta;
    float *mean, *rstd, *dgamma, *dbeta;
    float* parts;                      // [N][P][C][2]: forward mean and sum of squares about it, backward A and B, of a run of pixels
    float* sums;                       // [N][C][2]: A, B;  then [N][G][2]: s1 / M, s2 / M
    long long HW;
    int N, C, G, P;
    int chunks, lanes;                 // a pixel's chunks of VEC channels in one workgroup (team), and the pixels side by side in it
    int runs;                          // runs that `parts` holds (P of the launch that wrote it)
    int team;                          // a group per team: its threads
    int rows;                          // parameter gradients: rows of `sums` (N, or runs of images already summed up)
    float eps;
};

// VEC neighbouring channels of one pixel as they lie in memory, and their values
template <typename T, int VEC> struct Raw { typedef __attribute__((ext_vector_type(VEC * sizeof(T) / 4))) int type; };
template <> struct Raw<bf16raw, 1> { typedef bf16raw type; };
template <> struct Raw<bf16raw, 2> { typedef unsigned type; };
template <> struct Raw<float, 1> { typedef float type; };
template <typename T, int VEC> __device__ __forceinline__ typename Raw<T, VEC>::type vec_read(const T* p) { return *(const typename Raw<T, VEC>::type*)p; }
template <typename T, int VEC> __device__ __forceinline__ void vec_values(const typename Raw<T, VEC>::type& v, float* f) {
    if constexpr (VEC == 1) f[0] = Elem<T>::to_f32(v);
    else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = __int_as_float(v[e]);
    } else if constexpr (VEC == 2) {
        f[0] = __uint_as_float(v << 16);
        f[1] = __uint_as_float(v & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
            f[2 * e] = __uint_as_float((unsigned)v[e] << 16);
            f[2 * e + 1] = __uint_as_float((unsigned)v[e] & 0xFFFF0000u);
        }
    }
}
template <typename T, int VEC> __device__ __forceinline__ void vec_load(const T* p, float* f) { vec_values<T, VEC>(vec_read<T, VEC>(p), f); }
template <typename T, int VEC> __device__ __forceinline__ void vec_store(T* p, const float* f) {
    if constexpr (VEC == 1) Elem<T>::st(p, f[0]);
    else if constexpr (sizeof(T) == 4) {
        typedef __attribute__((ext_vector_type(VEC))) float V;
        V v;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = f[e];
        *(V*)p = v;
    } else if constexpr (VEC == 2) {
        *(int*)p = pack_bf16x2(f[0], f[1]);
    } else {
        typedef __attribute__((ext_vector_type(VEC / 2))) int V;
        V v;
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) v[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
        *(V*)p = v;
    }
}

// A workgroup takes a run of pixels of one image (and, where a pixel has more than 256 chunks, 256 of them): thread = (pixel lane,
// chunk), so that a thread keeps its channels and the workgroup reads whole pixels side by side.
#define GN_THREADS 256
#define GN_UNROLL 8
#define GN_JOIN_CHANNELS 512       // at most, where the apply kernels join the runs themselves
struct GnPlace { int n, run, chunk, lane, c; long long first, last; bool on; };        // c: first channel; pixels [first, last) of image n
template <int VEC> __device__ __forceinline__ GnPlace gn_place(const GnArgs& a) {
    GnPlace q;
    q.n = blockIdx.x / (unsigned)a.P;
    q.run = blockIdx.x - q.n * a.P;
    q.lane = threadIdx.x / a.chunks;
    q.chunk = threadIdx.x - q.lane * a.chunks;
    q.c = (blockIdx.y * a.chunks + q.chunk) * VEC;
    q.on = q.lane < a.lanes && q.c < a.C;
    const long long per = (a.HW + a.P - 1) / a.P;
    q.first = q.run * per;
    q.last = q.first + per < a.HW ? q.first + per : a.HW;
    return q;
}

// Mean, sum of squares about it and count of two sets of values as those of their union
__device__ __forceinline__ void gn_join(float& mean, float& m2, float& n, float omean, float om2, float on) {
    const float all = n + on;
    if (all > 0.f) {
        const float d = omean - mean, w = on / all;
        mean = fmaf(d, w, mean);
        m2 += om2 + d * d * (n * w);
        n = all;
    }
}

// The pixel lanes of a workgroup joined in halves: lane 0 has its channels' mean and sum of squares over all lanes
template <int VEC>
__device__ __forceinline__ void gn_join_lanes(const GnArgs& a, const GnPlace& q, float* mean, float* m2, float& n, float (*sh)[VEC][GN_THREADS], float* shn) {
    for (int have = a.lanes; have > 1;) {
        const int keep = (have + 1) / 2;
        __syncthreads();
        if (q.on && q.lane >= keep && q.lane < have) {
            shn[threadIdx.x] = n;
#pragma unroll
            for (int e = 0; e < VEC; ++e) { sh[0][e][threadIdx.x] = mean[e]; sh[1][e][threadIdx.x] = m2[e]; }
        }
        __syncthreads();
        if (q.on && q.lane + keep < have) {
            const int o = threadIdx.x + keep * a.chunks;
            const float on = shn[o], all = n + on, w = all > 0.f ? on / all : 0.f, nw = n * w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = sh[0][e][o] - mean[e];
                mean[e] = fmaf(d, w, mean[e]);
                m2[e] += sh[1][e][o] + d * d * nw;
            }
            n = all;
        }
        have = keep;
    }
}
// ... added in halves
template <int VEC>
__device__ __forceinline__ void gn_add_lanes(const GnArgs& a, const GnPlace& q, float* s, float* r, float (*sh)[VEC][GN_THREADS]) {
    for (int have = a.lanes; have > 1;) {
        const int keep = (have + 1) / 2;
        __syncthreads();
        if (q.on && q.lane >= keep && q.lane < have) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) { sh[0][e][threadIdx.x] = s[e]; sh[1][e][threadIdx.x] = r[e]; }
        }
        __syncthreads();
        if (q.on && q.lane + keep < have) {
            const int o = threadIdx.x + keep * a.chunks;
#pragma unroll
            for (int e = 0; e < VEC; ++e) { s[e] += sh[0][e][o]; r[e] += sh[1][e][o]; }
        }
        have = keep;
    }
}

// Forward statistics of a run of pixels (8 x 524288 x 16 bf16: 39 us).  A thread sums 4 pixels of a channel, then their squares about their own mean, and joins
// that to what it has: no shift has to be guessed and no large squares cancel.
template <typename T, int VEC>
__global__ __launch_bounds__(GN_THREADS) void gn_stats_kernel(const GnArgs a) {
    __shared__ float sh[2][VEC][GN_THREADS], shn[GN_THREADS];
    const GnPlace q = gn_place<VEC>(a);
    const T* x = (const T*)a.x + (long long)q.n * a.HW * a.C + q.c;
    float mean[VEC], m2[VEC], n = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) mean[e] = m2[e] = 0.f;
    if (q.on) {
        constexpr int U = 4;
        long long p = q.first + q.lane;
        typename Raw<T, VEC>::type raw[U];
        auto whole = [&](long long at) { return at + (U - 1) * a.lanes < q.last; };
        auto fetch = [&](long long at) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = vec_read<T, VEC>(x + (at + u * a.lanes) * a.C);
        };
        if (whole(p)) fetch(p);
        for (; whole(p); p += U * a.lanes) {
            float f[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) vec_values<T, VEC>(raw[u], f[u]);
            if (whole(p + U * a.lanes)) fetch(p + U * a.lanes);        // on its way while this set is worked on
            const float all = n + U, w = U / all, nw = n * w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float s = 0.f, r = 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) s += f[u][e];
                s *= 1.f / U;
#pragma unroll
                for (int u = 0; u < U; ++u) r = fmaf(f[u][e] - s, f[u][e] - s, r);
                const float d = s - mean[e];
                mean[e] = fmaf(d, w, mean[e]);
                m2[e] += r + d * d * nw;
            }
            n = all;
        }
        for (; p < q.last; p += a.lanes) {
            float f[VEC];
            vec_load<T, VEC>(x + p * a.C, f);
            const float w = 1.f / (n + 1.f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = f[e] - mean[e];
                mean[e] = fmaf(d, w, mean[e]);
                m2[e] = fmaf(d * d, n * w, m2[e]);
            }
            n += 1.f;
        }
    }
    gn_join_lanes<VEC>(a, q, mean, m2, n, sh, shn);
    if (q.on && q.lane == 0) {
        float* out = a.parts + 2 * (((long long)q.n * a.P + q.run) * a.C + q.c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { out[2 * e] = mean[e]; out[2 * e + 1] = m2[e]; }
    }
}

// One workgroup per (image, group): the group's channels and runs of pixels joined to its mean and 1 / sqrt(var + eps)
__global__ __launch_bounds__(1024) void gn_finalize_kernel(const GnArgs a) {
    __shared__ float sh[3][16];
    for (long long at = blockIdx.x; at < (long long)a.N * a.G; at += gridDim.x) {
        const int n = (unsigned)at / (unsigned)a.G, g = (unsigned)at % (unsigned)a.G, cpg = a.C / a.G;
        const long long per = (a.HW + a.runs - 1) / a.runs;
        float mean = 0.f, m2 = 0.f, count = 0.f;
        for (long long i = threadIdx.x; i < (long long)a.runs * cpg; i += 1024) {
            const long long p = i / cpg, c = g * cpg + (i - p * cpg), left = a.HW - p * per;
            const float2 v = *(const float2*)(a.parts + 2 * (((long long)n * a.runs + p) * a.C + c));
            gn_join(mean, m2, count, v.x, v.y, left <= 0 ? 0.f : (float)(left < per ? left : per));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) gn_join(mean, m2, count, __shfl_xor(mean, o, 64), __shfl_xor(m2, o, 64), __shfl_xor(count, o, 64));
        if ((threadIdx.x & 63) == 0) { sh[0][threadIdx.x >> 6] = mean; sh[1][threadIdx.x >> 6] = m2; sh[2][threadIdx.x >> 6] = count; }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 16; ++w) gn_join(mean, m2, count, sh[0][w], sh[1][w], sh[2][w]);
            a.mean[at] = mean;
            a.rstd[at] = 1.f / sqrtf(m2 / ((float)a.HW * cpg) + a.eps);
        }
        __syncthreads();                                               // the next group's values come to the same place
    }
}

// A thread's channels: mean, rstd gamma and beta of each
template <int VEC>
__device__ __forceinline__ void gn_channels(const GnArgs& a, const GnPlace& q, float* mean, float* scale, float* beta) {
    const int cpg = a.C / a.G;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const int c = q.c + e, g = c / cpg;
        mean[e] = a.mean[(long long)q.n * a.G + g];
        scale[e] = a.rstd[(long long)q.n * a.G + g] * (a.gamma ? a.gamma[c] : 1.f);
        beta[e] = a.beta ? a.beta[c] : 0.f;
    }
}

// The same from the runs, where a workgroup has all of an image's channels: its threads join their channels' runs, and each then goes
// over the channels of its groups.  All channels count the same pixels: a group's mean is the mean of theirs, its sum of squares that
// of theirs and of HW times the squares of their distances.
template <int VEC>
__device__ __forceinline__ void gn_channels_from_runs(const GnArgs& a, const GnPlace& q, float* mean, float* scale, float* beta, float (*sh)[VEC][GN_THREADS],
                                                      float* shn, float (*channel)[GN_JOIN_CHANNELS]) {
    float m2[VEC], n = 0.f;
    const long long per = (a.HW + a.runs - 1) / a.runs;
#pragma unroll
    for (int e = 0; e < VEC; ++e) mean[e] = m2[e] = 0.f;
    if (q.on)
        for (int p = q.lane; p < a.runs; p += a.lanes) {
            const float* v = a.parts + 2 * (((long long)q.n * a.runs + p) * a.C + q.c);
            const long long left = a.HW - p * per;
            const float on = left <= 0 ? 0.f : (float)(left < per ? left : per), all = n + on, w = all > 0.f ? on / all : 0.f, nw = n * w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = v[2 * e] - mean[e];
                mean[e] = fmaf(d, w, mean[e]);
                m2[e] += v[2 * e + 1] + d * d * nw;
            }
            n = all;
        }
    gn_join_lanes<VEC>(a, q, mean, m2, n, sh, shn);
    if (q.on && q.lane == 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) { channel[0][q.c + e] = mean[e]; channel[1][q.c + e] = m2[e]; }
    }
    __syncthreads();
    if (!q.on) return;
    const int cpg = a.C / a.G;
    int have = -1;
    float gmean = 0.f, rstd = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const int c = q.c + e, g = c / cpg;
        if (g != have) {
            float s = 0.f, d = 0.f;
            for (int j = g * cpg; j < (g + 1) * cpg; ++j) s += channel[0][j];
            gmean = s / (float)cpg;
            for (int j = g * cpg; j < (g + 1) * cpg; ++j) d += channel[1][j] + (float)a.HW * (channel[0][j] - gmean) * (channel[0][j] - gmean);
            rstd = 1.f / sqrtf(d / ((float)a.HW * cpg) + a.eps);
            have = g;
            if (q.run == 0 && q.lane == 0 && c == g * cpg) {
                a.mean[(long long)q.n * a.G + g] = gmean;
                a.rstd[(long long)q.n * a.G + g] = rstd;
            }
        }
        mean[e] = gmean;
        scale[e] = rstd * (a.gamma ? a.gamma[c] : 1.f);
        beta[e] = a.beta ? a.beta[c] : 0.f;
    }
}

template <typename T, int VEC, int ACT, bool JOINED>
__global__ __launch_bounds__(GN_THREADS) void gn_apply_kernel(const GnArgs a) {
    constexpr int U = 4;
    const GnPlace q = gn_place<VEC>(a);
    const T* x = (const T*)a.x + (long long)q.n * a.HW * a.C + q.c;
    T* y = (T*)a.y + (long long)q.n * a.HW * a.C + q.c;
    float mean[VEC], scale[VEC], beta[VEC];
    if constexpr (JOINED) {
        if (!q.on) return;
        gn_channels<VEC>(a, q, mean, scale, beta);
    } else {
        __shared__ float sh[2][VEC][GN_THREADS], shn[GN_THREADS], channel[2][GN_JOIN_CHANNELS];
        gn_channels_from_runs<VEC>(a, q, mean, scale, beta, sh, shn, channel);
        if (!q.on) return;
    }
    // whole sets of loads first, without a branch between a load and what takes its value apart; then one by one
    auto set = [&](long long p, auto count) {
        constexpr int N = decltype(count)::value;
        float f[N][VEC];
#pragma unroll
        for (int u = 0; u < N; ++u) vec_load<T, VEC>(x + (p + u * a.lanes) * a.C, f[u]);
#pragma unroll
        for (int u = 0; u < N; ++u) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[u][e] = gn_act<ACT>(gn_u(f[u][e], mean[e], scale[e], beta[e]));
            vec_store<T, VEC>(y + (p + u * a.lanes) * a.C, f[u]);
        }
    };
    long long p = q.first + q.lane;
    for (; p + (U - 1) * a.lanes < q.last; p += U * a.lanes) set(p, Int<U>());
    for (; p < q.last; p += a.lanes) set(p, Int<1>());
}

// Backward sums A, B of a run of pixels (8 x 524288 x 16 bf16: 58 us; 66 without the loads of the next set ahead)
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_sums_kernel(const GnArgs a) {
    constexpr int U = 4;
    __shared__ float sh[2][VEC][GN_THREADS];
    const GnPlace q = gn_place<VEC>(a);
    const long long at = (long long)q.n * a.HW * a.C + q.c;
    const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
    float s[VEC], r[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = r[e] = 0.f;
    if (q.on) {
        float mean[VEC], scale[VEC], beta[VEC];
        gn_channels<VEC>(a, q, mean, scale, beta);
        typename Raw<T, VEC>::type rx[U], ry[U];
        auto whole = [&](long long at) { return at + (U - 1) * a.lanes < q.last; };
        auto fetch = [&](long long at) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = vec_read<T, VEC>(x + (at + u * a.lanes) * a.C);
                ry[u] = vec_read<T, VEC>(dy + (at + u * a.lanes) * a.C);
            }
        };
        auto add = [&](const float* f, const float* d, float* ls, float* lr) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float du = d[e] * gn_slope<ACT>(gn_u(f[e], mean[e], scale[e], beta[e]));
                ls[e] += du;
                lr[e] = fmaf(du, f[e] - mean[e], lr[e]);
            }
        };
        long long p = q.first + q.lane;
        if (whole(p)) fetch(p);
        for (; whole(p); p += U * a.lanes) {
            float f[U][VEC], d[U][VEC], ls[VEC], lr[VEC];              // these few first: shorter chains of roundings
#pragma unroll
            for (int e = 0; e < VEC; ++e) ls[e] = lr[e] = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) { vec_values<T, VEC>(rx[u], f[u]); vec_values<T, VEC>(ry[u], d[u]); }
            if (whole(p + U * a.lanes)) fetch(p + U * a.lanes);        // on its way while this set is worked on
#pragma unroll
            for (int u = 0; u < U; ++u) add(f[u], d[u], ls, lr);
#pragma unroll
            for (int e = 0; e < VEC; ++e) { s[e] += ls[e]; r[e] += lr[e]; }
        }
        for (; p < q.last; p += a.lanes) {
            float f[VEC], d[VEC];
            vec_load<T, VEC>(x + p * a.C, f);
            vec_load<T, VEC>(dy + p * a.C, d);
            add(f, d, s, r);
        }
        const int cpg = a.C / a.G;
#pragma unroll
        for (int e = 0; e < VEC; ++e) r[e] *= a.rstd[(long long)q.n * a.G + (q.c + e) / cpg];
    }
    gn_add_lanes<VEC>(a, q, s, r, sh);
    if (q.on && q.lane == 0) {
        float* out = a.parts + 2 * (((long long)q.n * a.P + q.run) * a.C + q.c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { out[2 * e] = s[e]; out[2 * e + 1] = r[e]; }
    }
}

// One workgroup per (image, group): A and B of its channels over the runs of pixels, s1 / M and s2 / M over the channels.  Threads are
// (run lane, channel) with the channels side by side in memory; 1024 channels at a time.
__global__ __launch_bounds__(1024) void gn_bwd_finalize_kernel(const GnArgs a) {
    __shared__ double sh[2][1024];
    for (long long at = blockIdx.x; at < (long long)a.N * a.G; at += gridDim.x) {
        const int n = (unsigned)at / (unsigned)a.G, g = (unsigned)at % (unsigned)a.G, cpg = a.C / a.G;
        const int side = cpg < 1024 ? cpg : 1024, lanes = 1024 / side, lane = threadIdx.x / side, j = threadIdx.x - lane * side;
        double s1 = 0, s2 = 0;
        for (int c0 = 0; c0 < cpg; c0 += side) {
            const int c = g * cpg + c0 + j;
            const bool on = lane < lanes && c0 + j < cpg;
            double p = 0, r = 0;
            if (on)
                for (int i = lane; i < a.runs; i += lanes) {
                    const float2 v = *(const float2*)(a.parts + 2 * (((long long)n * a.runs + i) * a.C + c));
                    p += v.x;
                    r += v.y;
                }
            for (int have = lanes; have > 1;) {
                const int keep = (have + 1) / 2;
                __syncthreads();
                if (lane >= keep && lane < have) { sh[0][threadIdx.x] = p; sh[1][threadIdx.x] = r; }
                __syncthreads();
                if (lane + keep < have) { p += sh[0][threadIdx.x + keep * side]; r += sh[1][threadIdx.x + keep * side]; }
                have = keep;
            }
            if (on && lane == 0) {
                a.sums[2 * ((long long)n * a.C + c)] = (float)p;
                a.sums[2 * ((long long)n * a.C + c) + 1] = (float)r;
                const double gamma = a.gamma ? a.gamma[c] : 1.f;
                s1 += gamma * p;
                s2 += gamma * r;
            }
        }
        __syncthreads();
        sh[0][threadIdx.x] = s1;
        sh[1][threadIdx.x] = s2;
        for (int o = 512; o > 0; o >>= 1) {
            __syncthreads();
            if ((int)threadIdx.x < o) { sh[0][threadIdx.x] += sh[0][threadIdx.x + o]; sh[1][threadIdx.x] += sh[1][threadIdx.x + o]; }
        }
        if (threadIdx.x == 0) {
            const double m = (double)a.HW * cpg;
            float* out = a.sums + 2 * (long long)a.N * a.C + 2 * at;
            out[0] = (float)(sh[0][0] / m);
            out[1] = (float)(sh[1][0] / m);
        }
        __syncthreads();                                               // the next group's values come to the same place
    }
}

// dbeta = sum A and dgamma = sum B over rows [C][2] of images or runs: 16 channels a workgroup, 16 row lanes with 4 loads in flight each
#define GN_SIDE 16
__device__ __forceinline__ void gn_row_sums(const float* sums, long long first, long long last, int C, int c, double (*sh)[GN_THREADS], double& p, double& r) {
    constexpr int LANES = GN_THREADS / GN_SIDE;
    p = r = 0;
    if (c < C) {
        long long n = first + threadIdx.x / GN_SIDE;
        for (; n + 3 * LANES < last; n += 4 * LANES) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = *(const float2*)(sums + 2 * ((n + u * LANES) * C + c));
#pragma unroll
            for (int u = 0; u < 4; ++u) { p += v[u].x; r += v[u].y; }
        }
        for (; n < last; n += LANES) {
            const float2 v = *(const float2*)(sums + 2 * (n * C + c));
            p += v.x;
            r += v.y;
        }
    }
    sh[0][threadIdx.x] = p;
    sh[1][threadIdx.x] = r;
    for (int o = GN_THREADS / 2; o >= GN_SIDE; o /= 2) {
        __syncthreads();
        if ((int)threadIdx.x < o) { sh[0][threadIdx.x] += sh[0][threadIdx.x + o]; sh[1][threadIdx.x] += sh[1][threadIdx.x + o]; }
    }
    p = sh[0][threadIdx.x];
    r = sh[1][threadIdx.x];
}
__device__ __forceinline__ void gn_param_grads(const GnArgs& a, const float* sums, int block, double (*sh)[GN_THREADS]) {
    const int c = block * GN_SIDE + (threadIdx.x % GN_SIDE);
    double p, r;
    gn_row_sums(sums, 0, a.rows, a.C, c, sh, p, r);
    if (threadIdx.x < GN_SIDE && c < a.C) {
        if (a.dbeta) a.dbeta[c] = (float)p;
        if (a.dgamma) a.dgamma[c] = (float)r;
    }
}
__global__ __launch_bounds__(GN_THREADS) void gn_param_grads_kernel(const GnArgs a, const float* sums) {
    __shared__ double sh[2][GN_THREADS];
    gn_param_grads(a, sums, blockIdx.x, sh);
}
// ... of many images: runs of them first, to rows of `out`
__global__ __launch_bounds__(GN_THREADS) void gn_image_runs_kernel(const GnArgs a, float* out) {
    __shared__ double sh[2][GN_THREADS];
    const int c = blockIdx.x * GN_SIDE + (threadIdx.x % GN_SIDE);
    const long long per = (a.N + (long long)gridDim.y - 1) / gridDim.y, first = blockIdx.y * per, last = first + per < a.N ? first + per : a.N;
    double p, r;
    gn_row_sums(a.sums, first, last, a.C, c, sh, p, r);
    if (threadIdx.x < GN_SIDE && c < a.C) {
        out[2 * ((long long)blockIdx.y * a.C + c)] = (float)p;
        out[2 * ((long long)blockIdx.y * a.C + c) + 1] = (float)r;
    }
}

// s1 / M and s2 / M of a thread's channels from the runs, as gn_channels_from_runs
template <int VEC>
__device__ __forceinline__ void gn_sums_from_runs(const GnArgs& a, const GnPlace& q, float* k1, float* k2, float (*sh)[VEC][GN_THREADS],
                                                  float (*channel)[GN_JOIN_CHANNELS]) {
    float s[VEC], r[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = r[e] = 0.f;
    if (q.on)
        for (int p = q.lane; p < a.runs; p += a.lanes) {
            const float* v = a.parts + 2 * (((long long)q.n * a.runs + p) * a.C + q.c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) { s[e] += v[2 * e]; r[e] += v[2 * e + 1]; }
        }
    gn_add_lanes<VEC>(a, q, s, r, sh);
    if (q.on && q.lane == 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float gamma = a.gamma ? a.gamma[q.c + e] : 1.f;
            channel[0][q.c + e] = gamma * s[e];
            channel[1][q.c + e] = gamma * r[e];
        }
    }
    __syncthreads();
    if (!q.on) return;
    const int cpg = a.C / a.G;
    const float m = (float)a.HW * cpg;
    int have = -1;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const int g = (q.c + e) / cpg;
        if (g != have) {
            s1 = s2 = 0.f;
            for (int j = g * cpg; j < (g + 1) * cpg; ++j) { s1 += channel[0][j]; s2 += channel[1][j]; }
            s1 /= m;
            s2 /= m;
            have = g;
        }
        k1[e] = s1;
        k2[e] = s2;
    }
}

// dx; and, by the workgroups behind those of the last run, the parameter gradients
template <typename T, int VEC, int ACT, bool JOINED>
__global__ __launch_bounds__(GN_THREADS) void gn_bwd_apply_kernel(const GnArgs a) {
    constexpr int U = 4;
    if (blockIdx.x >= (unsigned)(a.N * a.P)) {
        __shared__ double sh[2][GN_THREADS];
        if (blockIdx.y) return;
        gn_param_grads(a, JOINED ? a.sums : a.parts, (int)(blockIdx.x - (unsigned)(a.N * a.P)), sh);
        return;
    }
    const GnPlace q = gn_place<VEC>(a);
    const long long at = (long long)q.n * a.HW * a.C + q.c;
    const T *x = (const T*)a.x + at, *dy = (const T*)a.dy + at;
    T* dx = (T*)a.dx + at;
    float mean[VEC], scale[VEC], beta[VEC], k1[VEC], k2[VEC];          // dx = scale du - k1 - (x - mean) k2
    const int cpg = a.C / a.G;
    if constexpr (JOINED) {
        if (!q.on) return;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float2 m = *(const float2*)(a.sums + 2 * (long long)a.N * a.C + 2 * ((long long)q.n * a.G + (q.c + e) / cpg));
            k1[e] = m.x;
            k2[e] = m.y;
        }
    } else {
        __shared__ float sh[2][VEC][GN_THREADS], channel[2][GN_JOIN_CHANNELS];
        gn_sums_from_runs<VEC>(a, q, k1, k2, sh, channel);
        if (!q.on) return;
    }
    gn_channels<VEC>(a, q, mean, scale, beta);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const float rstd = a.rstd[(long long)q.n * a.G + (q.c + e) / cpg];
        k1[e] *= rstd;
        k2[e] *= rstd * rstd;
    }
    auto set = [&](long long p, auto count) {
        constexpr int N = decltype(count)::value;
        float f[N][VEC], d[N][VEC];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            vec_load<T, VEC>(x + (p + u * a.lanes) * a.C, f[u]);
            vec_load<T, VEC>(dy + (p + u * a.lanes) * a.C, d[u]);
        }
#pragma unroll
        for (int u = 0; u < N; ++u) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float du = d[u][e] * gn_slope<ACT>(gn_u(f[u][e], mean[e], scale[e], beta[e]));
                d[u][e] = fmaf(scale[e], du, -fmaf(f[u][e] - mean[e], k2[e], k1[e]));
            }
            vec_store<T, VEC>(dx + (p + u * a.lanes) * a.C, d[u]);
        }
    };
    long long p = q.first + q.lane;
    for (; p + (U - 1) * a.lanes < q.last; p += U * a.lanes) set(p, Int<U>());
    for (; p < q.last; p += a.lanes) set(p, Int<1>());
}

// ------------------------------------------------------------------------------------------------ a whole group in registers
// Where the values of one (image, group) fit the registers of a team of 8 or 64 lanes or of a workgroup, KEEP of them per thread, x
// (and dy) are read once and one launch does it all: 512 x 128 in 8 groups bf16 7 us forward, bound by its latency; 64 x 4096 x 64 in 8
// groups fp32 27 us, 4.9 TB/s.  Threads are (pixel lane, chunk of VEC channels of the group).  Neighbouring
// groups, which share cache lines, go to one XCD: workgroups are dealt to the 8 XCDs in turn.
#define GN_KEEP 32
struct GnGroup { int n, g, c, tid, lane; long long at; bool on; };          // c: first channel; at: its place in the image's first pixel of the lane
template <int VEC> __device__ __forceinline__ GnGroup gn_group(const GnArgs& a) {
    GnGroup q;
    const unsigned teams = blockDim.x / a.team, id = ((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) * teams + threadIdx.x / a.team;
    q.tid = threadIdx.x % a.team;
    q.n = id / (unsigned)a.G;
    q.g = id - q.n * a.G;
    q.lane = q.tid / a.chunks;
    q.c = q.g * (a.C / a.G) + (q.tid - q.lane * a.chunks) * VEC;
    q.on = q.n < a.N && q.lane < a.lanes;
    q.at = ((long long)q.n * a.HW + q.lane) * a.C + q.c;
    return q;
}

// Sum over the team; every thread gets it
__device__ __forceinline__ float gn_total(float v, float* sh, int team) {
    v += __shfl_xor(v, 1, 64);
    v += __shfl_xor(v, 2, 64);
    v += __shfl_xor(v, 4, 64);
    if (team == 8) return v;
    v += __shfl_xor(v, 8, 64);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    if (team == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) s += sh[w];
    return s;
}
__device__ __forceinline__ void gn_sync(int team) {
    if (team > 64) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(1024) void gn_group_fwd_kernel(const GnArgs a) {
    constexpr int R = GN_KEEP / VEC;
    __shared__ float sh[16];
    const GnGroup q = gn_group<VEC>(a);
    const T* x = (const T*)a.x + q.at;
    typename Raw<T, VEC>::type raw[R];                                 // taken apart after all loads are on their way
    float f[R][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        raw[r] = typename Raw<T, VEC>::type{};
        if (q.on && q.lane + r * a.lanes < a.HW) raw[r] = vec_read<T, VEC>(x + (long long)r * a.lanes * a.C);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) vec_values<T, VEC>(raw[r], f[r]);
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s += f[r][e];
    const float m = (float)(a.HW * (a.C / a.G)), mean = gn_total(s, sh, a.team) / m;
    s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (q.on && q.lane + r * a.lanes < a.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) s = fmaf(f[r][e] - mean, f[r][e] - mean, s);
        }
    const float rstd = 1.f / sqrtf(gn_total(s, sh, a.team) / m + a.eps);
    if (q.on && q.tid == 0) { a.mean[(long long)q.n * a.G + q.g] = mean; a.rstd[(long long)q.n * a.G + q.g] = rstd; }
    if (!q.on) return;
    float scale[VEC], beta[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        scale[e] = rstd * (a.gamma ? a.gamma[q.c + e] : 1.f);
        beta[e] = a.beta ? a.beta[q.c + e] : 0.f;
    }
    T* y = (T*)a.y + q.at;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (q.lane + r * a.lanes < a.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[r][e] = gn_act<ACT>(gn_u(f[r][e], mean, scale[e], beta[e]));
            vec_store<T, VEC>(y + (long long)r * a.lanes * a.C, f[r]);
        }
}

// dx, and A and B of the group's channels; gn_param_grads_kernel sums those over the images
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(1024) void gn_group_bwd_kernel(const GnArgs a) {
    constexpr int R = GN_KEEP / VEC;
    __shared__ float sh[16];
    extern __shared__ float part[];                                    // [2][VEC][threads]
    const GnGroup q = gn_group<VEC>(a);
    const T *x = (const T*)a.x + q.at, *dy = (const T*)a.dy + q.at;
    const float mean = q.on ? a.mean[(long long)q.n * a.G + q.g] : 0.f, rstd = q.on ? a.rstd[(long long)q.n * a.G + q.g] : 0.f;
    typename Raw<T, VEC>::type fraw[R], draw[R];
    float f[R][VEC], d[R][VEC], gamma[VEC], beta[VEC], p[VEC], s[VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        fraw[r] = draw[r] = typename Raw<T, VEC>::type{};
        if (q.on && q.lane + r * a.lanes < a.HW) {
            fraw[r] = vec_read<T, VEC>(x + (long long)r * a.lanes * a.C);
            draw[r] = vec_read<T, VEC>(dy + (long long)r * a.lanes * a.C);
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        gamma[e] = q.on && a.gamma ? a.gamma[q.c + e] : 1.f;
        beta[e] = q.on && a.beta ? a.beta[q.c + e] : 0.f;
        p[e] = s[e] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        vec_values<T, VEC>(fraw[r], f[r]);
        vec_values<T, VEC>(draw[r], d[r]);
        if (q.on && q.lane + r * a.lanes < a.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                d[r][e] *= gn_slope<ACT>(gn_u(f[r][e], mean, rstd * gamma[e], beta[e]));
                f[r][e] = (f[r][e] - mean) * rstd;
                p[e] += d[r][e];
                s[e] = fmaf(d[r][e], f[r][e], s[e]);
            }
        }
    }
    for (int have = a.lanes; have > 1;) {
        const int keep = (have + 1) / 2;
        gn_sync(a.team);
        if (q.on && q.lane >= keep && q.lane < have) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) { part[e * blockDim.x + threadIdx.x] = p[e]; part[(VEC + e) * blockDim.x + threadIdx.x] = s[e]; }
        }
        gn_sync(a.team);
        if (q.on && q.lane + keep < have) {
            const int o = threadIdx.x + keep * a.chunks;
#pragma unroll
            for (int e = 0; e < VEC; ++e) { p[e] += part[e * blockDim.x + o]; s[e] += part[(VEC + e) * blockDim.x + o]; }
        }
        have = keep;
    }
    float g1 = 0.f, g2 = 0.f;
    if (q.on && q.lane == 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float* out = a.sums + 2 * ((long long)q.n * a.C + q.c + e);
            out[0] = p[e];
            out[1] = s[e];
            g1 = fmaf(gamma[e], p[e], g1);
            g2 = fmaf(gamma[e], s[e], g2);
        }
    }
    const float m = (float)(a.HW * (a.C / a.G));
    g1 = gn_total(g1, sh, a.team) / m;
    g2 = gn_total(g2, sh, a.team) / m;
    if (!q.on) return;
    T* dx = (T*)a.dx + q.at;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (q.lane + r * a.lanes < a.HW) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[r][e] = rstd * (gamma[e] * d[r][e] - fmaf(f[r][e], g2, g1));
            vec_store<T, VEC>(dx + (long long)r * a.lanes * a.C, d[r]);
        }
}

static inline bool gn_shape_ok(int dtype, int N, long long HW, int C, int groups, int act) {
    return (dtype == ERF_F32 || dtype == ERF_BF16) && N > 0 && N <= (1 << 23) && HW > 0 && C > 0 && groups > 0 && C % groups == 0 && act >= 0 &&
           act <= 2 && (long long)N * groups <= 0x7FFFFFFFll && C <= (1 << 20) && HW <= (1ll << 40) / C;
}

// Channels per access: the most that divide C, fit 16 bytes and lie on their boundaries
static inline int gn_vec(int dtype, int C, unsigned long long addresses) {
    const int size = dtype == ERF_BF16 ? 2 : 4;
    int v = 16 / size;
    while (v > 1 && (C % v || addresses % (v * size))) v /= 2;
    return v;
}
// Runs of pixels per image: about 1024 workgroups in all (512 to 4096 are within 5 % of each other on large maps), each thread with `each`
// pixels at least (8: 6 x 32768 x 64 bf16 25 / 39 us forward / backward, with 4 in the apply kernels 27 / 45; 3 x 5673 x 30 10.4 / 10.2
// against 9.9 / 9.7), at most `most` runs
#define GN_MAX_RUNS 512
template <int VEC> static inline dim3 gn_plan(GnArgs& a, int each, int most) {
    const int chunks = a.C / VEC;
    a.chunks = chunks < GN_THREADS ? chunks : GN_THREADS;
    a.lanes = GN_THREADS / a.chunks;
    const int slabs = (chunks + a.chunks - 1) / a.chunks;
    const long long images = (long long)a.N * slabs, want = (1024 + images - 1) / images, full = (a.HW + (long long)a.lanes * each - 1) / ((long long)a.lanes * each);
    const long long p = want < full ? want : full;
    a.P = (int)(p < 1 ? 1 : p > most ? most : p);
    return dim3((unsigned)a.P * (unsigned)a.N, (unsigned)slabs);
}

// The plan of a group per team: channels per access (the most that divide a group) and the smallest team that has the values in
// registers and either fills the chip with threads or leaves each thread one access.  A group per team saves launches; by runs of
// pixels the memory is read better, the more so the less of each cache line is one group's.  So a group per team up to so many
// values of a group, which one workgroup works off alone, and up to so many pieces (a pixel's channels of one group); in all
// sizes of small groups, and for more images than runs are good for.  Group against runs, us, forward at 16 bytes an access: 64 x 4096 x 64 in 8 groups bf16 24 / 28, twice
// the pixels 43 / 43; 64 x 1024 x 128 in 32 fp32 24 / 23, twice 43 / 38; 3 channels a group: 64 x 1024 x 48 bf16 16 / 20, fp32 19 / 18,
// twice 26 / 24 and 30 / 22; few large groups: 1 x 2048 x 48 in 16 10 / 16, 3 x 5673 x 30 in 6 15 / 10.  Backward, bf16: 64 x 1024 x 64
// in 8 19 / 20, twice 36 / 29; 1 x 1024 x 64 in 8 13 / 15, twice 15 / 15; 16 x 2048 x 64 in 16 17 / 18; fp32: 1 x 512 x 64 in 8 11 / 10, 1 x
// 2048 x 64 in 16 13 / 10, 512 x 64 x 128 in 16 22 / 24; 1024 x 512 x 48 in 16 bf16 123 / 62, 4096 x 128 x 64 in 8 90 / 376.
static bool gn_group_plan(GnArgs& a, int dtype, unsigned long long addresses, int& vec, bool backward) {
    const int cpg = a.C / a.G;
    vec = gn_vec(dtype, cpg, addresses);
    a.chunks = cpg / vec;
    const long long groups = (long long)a.N * a.G;
    const bool bf16 = dtype == ERF_BF16, wide = vec * (bf16 ? 2 : 4) == 16;
    const long long values = a.HW * cpg, pieces = groups * a.HW;
    if (backward ? values > (bf16 ? 8192 : 4096) : wide ? a.HW > 4096 : values > 8192) return false;
    if (pieces > (backward ? 1 << 19 : wide ? 1 << 21 : 1 << 20) && a.N <= 1024 && values > 512) return false;
    for (a.team = 8; a.team <= 1024; a.team = a.team == 8 ? 64 : 4 * a.team) {
        a.lanes = a.team / a.chunks;
        if (a.lanes && a.HW <= (long long)a.lanes * GN_KEEP / vec && groups * a.team < 1ll << 31 && (a.team == 1024 || groups * a.team >= (1 << 17) || a.HW <= a.lanes)) return true;
    }
    return false;
}
static inline dim3 gn_group_block(const GnArgs& a) { return dim3(a.team < 256 ? 256 : (unsigned)a.team); }
static inline dim3 gn_group_grid(const GnArgs& a) {
    const long long teams = gn_group_block(a).x / a.team, blocks = ((long long)a.N * a.G + teams - 1) / teams;
    return dim3((unsigned)((blocks + 7) / 8 * 8));
}
// Images summed up before the parameter gradients are: runs of at least 64
static inline int gn_image_runs(int N) { return N <= 256 ? 1 : N / 64 < 64 ? N / 64 : 64; }

template <typename T, int VEC, int ACT>
static void gn_group_fwd_launch(GnArgs a, hipStream_t s) {
    hipLaunchKernelGGL((gn_group_fwd_kernel<T, VEC, ACT>), gn_group_grid(a), gn_group_block(a), 0, s, a);
}
static void gn_param_grads_launch(GnArgs a, hipStream_t s) {
    if (!a.dgamma && !a.dbeta) return;
    const unsigned blocks = (unsigned)((a.C + GN_SIDE - 1) / GN_SIDE);
    const float* sums = a.sums;
    a.rows = gn_image_runs(a.N);
    if (a.rows > 1) {
        hipLaunchKernelGGL(gn_image_runs_kernel, dim3(blocks, (unsigned)a.rows), dim3(GN_THREADS), 0, s, a, a.parts);
        sums = a.parts;
    } else {
        a.rows = a.N;
    }
    hipLaunchKernelGGL(gn_param_grads_kernel, dim3(blocks), dim3(GN_THREADS), 0, s, a, sums);
}
template <typename T, int VEC, int ACT>
static void gn_group_bwd_launch(GnArgs a, hipStream_t s) {
    hipLaunchKernelGGL((gn_group_bwd_kernel<T, VEC, ACT>), gn_group_grid(a), gn_group_block(a), 2 * VEC * gn_group_block(a).x * sizeof(float), s, a);
    gn_param_grads_launch(a, s);
}

// Whether the apply kernels join the runs: that costs each of their workgroups a look at all runs of its image, and saves a launch
// (3 x 5673 x 30 forward / backward 10 / 10 us against 11 / 13, 2 x 100000 x 16 18 / 22 against 19 / 24; 6 x 8192 x 128 and larger alike)
static inline bool gn_join_in_apply(const GnArgs& a, dim3 grid) {
    return grid.y == 1 && a.C <= GN_JOIN_CHANNELS && a.C / a.G <= 128 && (long long)a.P * a.C <= 8192;
}

// A launch has less than 2^32 threads: the workgroups take several groups each where there are very many
static inline dim3 gn_finalize_grid(const GnArgs& a) {
    const long long groups = (long long)a.N * a.G;
    return dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20));
}

template <typename T, int VEC, int ACT>
static void gn_fwd_launch(GnArgs a, hipStream_t s) {
    dim3 grid = gn_plan<VEC>(a, GN_UNROLL, GN_MAX_RUNS);
    hipLaunchKernelGGL((gn_stats_kernel<T, VEC>), grid, dim3(GN_THREADS), 0, s, a);
    const bool join = gn_join_in_apply(a, grid);
    a.runs = a.P;
    if (!join) hipLaunchKernelGGL(gn_finalize_kernel, gn_finalize_grid(a), dim3(1024), 0, s, a);
    grid = gn_plan<VEC>(a, GN_UNROLL, 1 << 20);
    if (join) hipLaunchKernelGGL((gn_apply_kernel<T, VEC, ACT, false>), grid, dim3(GN_THREADS), 0, s, a);
    else hipLaunchKernelGGL((gn_apply_kernel<T, VEC, ACT, true>), grid, dim3(GN_THREADS), 0, s, a);
}

template <typename T, int VEC, int ACT>
static void gn_bwd_launch(GnArgs a, hipStream_t s) {
    dim3 grid = gn_plan<VEC>(a, GN_UNROLL, GN_MAX_RUNS);
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, VEC, ACT>), grid, dim3(GN_THREADS), 0, s, a);
    a.runs = a.P;
    // the parameter gradients come from the runs as they are where these are few, else from the images' sums
    const bool params = a.dgamma || a.dbeta, join = gn_join_in_apply(a, grid) && (!params || (long long)a.N * a.runs <= 1024);
    if (!join) hipLaunchKernelGGL(gn_bwd_finalize_kernel, gn_finalize_grid(a), dim3(1024), 0, s, a);
    grid = gn_plan<VEC>(a, GN_UNROLL, 1 << 20);
    const bool few = params && (join || gn_image_runs(a.N) == 1);
    a.rows = join ? a.N * a.runs : a.N;
    if (few) grid.x += (unsigned)((a.C + GN_SIDE - 1) / GN_SIDE);
    if (join) hipLaunchKernelGGL((gn_bwd_apply_kernel<T, VEC, ACT, false>), grid, dim3(GN_THREADS), 0, s, a);
    else hipLaunchKernelGGL((gn_bwd_apply_kernel<T, VEC, ACT, true>), grid, dim3(GN_THREADS), 0, s, a);
    if (!few) gn_param_grads_launch(a, s);
}

#define GN_ACT(FN, T, VEC)                                                    \
    do {                                                                      \
        if (act == ERF_ACT_RELU) FN<T, VEC, ERF_ACT_RELU>(a, s);      \
        else if (act == ERF_ACT_SILU) FN<T, VEC, ERF_ACT_SILU>(a, s); \
        else FN<T, VEC, ERF_ACT_NONE>(a, s);                          \
    } while (0)
#define GN_PICK(FN)                                    \
    do {                                               \
        hipStream_t s = (hipStream_t)stream;           \
        if (dtype == ERF_F32) {                        \
            if (vec == 4) GN_ACT(FN, float, 4);        \
            else if (vec == 2) GN_ACT(FN, float, 2);   \
            else GN_ACT(FN, float, 1);                 \
        } else {                                       \
            if (vec == 8) GN_ACT(FN, bf16raw, 8);      \
            else if (vec == 4) GN_ACT(FN, bf16raw, 4); \
            else if (vec == 2) GN_ACT(FN, bf16raw, 2); \
            else GN_ACT(FN, bf16raw, 1);               \
        }                                              \
    } while (0)

extern "C" {

size_t erf_group_norm_workspace_bytes(int dtype, int N, long long HW, int C, int groups) {
    if (!gn_shape_ok(dtype, N, HW, C, groups, 0)) return 0;
    // the runs of pixels of any plan (which one depends on the addresses) or the runs of images, and the per-channel and per-group sums
    long long runs = (HW + GN_UNROLL - 1) / GN_UNROLL;
    const long long want = (1024 + N - 1) / N;
    runs = runs < want ? runs : want;
    runs = (runs < GN_MAX_RUNS ? runs : GN_MAX_RUNS) * N;
    runs = runs < gn_image_runs(N) ? gn_image_runs(N) : runs;
    return ((size_t)runs * C + (size_t)N * C + (size_t)N * groups) * 2 * sizeof(float);
}

int erf_group_norm_fwd(const void* x, void* y, int dtype, int N, long long HW, int C, int groups, const float* gamma, const float* beta,
                       float eps, int act, float* mean, float* rstd, void* workspace, void* stream) {
    if (!x || !y || !mean || !rstd || !workspace || !(eps >= 0) || !gn_shape_ok(dtype, N, HW, C, groups, act)) return ERF_EINVAL;
    GnArgs a = {};
    a.x = x; a.y = y; a.gamma = gamma; a.beta = beta; a.mean = mean; a.rstd = rstd; a.HW = HW; a.N = N; a.C = C; a.G = groups; a.eps = eps;
    a.sums = (float*)workspace;
    a.parts = a.sums + 2 * ((size_t)N * C + (size_t)N * groups);
    const unsigned long long addresses = (unsigned long long)x | (unsigned long long)y;
    int vec;
    if (gn_group_plan(a, dtype, addresses, vec, false)) {
        GN_PICK(gn_group_fwd_launch);
    } else {
        vec = gn_vec(dtype, C, addresses);
        GN_PICK(gn_fwd_launch);
    }
    return erf_check_launch();
}

int erf_group_norm_bwd(const void* x, const void* dy, void* dx, int dtype, int N, long long HW, int C, int groups, const float* gamma,
                       const float* beta, int act, const float* mean, const float* rstd, float* dgamma, float* dbeta, void* workspace,
                       void* stream) {
    if (!x || !dy || !dx || !mean || !rstd || !workspace || !gn_shape_ok(dtype, N, HW, C, groups, act)) return ERF_EINVAL;
    GnArgs a = {};
    a.x = x; a.dy = dy; a.dx = dx; a.gamma = gamma; a.beta = beta; a.mean = (float*)mean; a.rstd = (float*)rstd; a.dgamma = dgamma;
    a.dbeta = dbeta; a.HW = HW; a.N = N; a.C = C; a.G = groups;
    a.sums = (float*)workspace;
    a.parts = a.sums + 2 * ((size_t)N * C + (size_t)N * groups);
    const unsigned long long addresses = (unsigned long long)x | (unsigned long long)dy | (unsigned long long)dx;
    int vec;
    if (gn_group_plan(a, dtype, addresses, vec, true)) {
        GN_PICK(gn_group_bwd_launch);
    } else {
        vec = gn_vec(dtype, C, addresses);
        GN_PICK(gn_bwd_launch);
    }
    return erf_check_launch();
}

}  // extern "C"
