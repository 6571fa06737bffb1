// Log probabilities of given labels, entropy and the most probable classes, over the class axis of logits laid out as rows
// (classes side by side: tokens, classifier outputs, channels-last maps) or as planes (NCHW maps); and the gradient.
//
//     m = max z,  s = sum e^{z - m},  log p_j = (z_j - m) - log s,  H = log s - sum e^{z - m} (z - m) / s
//     dz_j = gl ([j = t] - p_j) - gh p_j (log p_j + H) + sum_k gk ([j = i_k] - p_j)
//
// One pass over the logits: running maximum, sum and weighted sum in fp32, rescaled where the maximum grows.  H is a sum of
// terms of one sign.  exp runs in base 2, (z - m) log2 e.  The backward pass takes m and log s apart: z - m is exact where it
// matters, while m + log s would lose log p's digits for logits far from 0.
//
// -inf logits have p = 0 and add nothing; a row without any finite logit, or with +inf or NaN, has no distribution: NaN.
#include "../../include/erfnet_mi355.h"
#include "common.cuh"

#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f

// running maximum, sum of 2^y and sum of 2^y y, y = (z - base) log2 e; base is m, or 0 while m is -inf
struct Stat { float m, s, t; };
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void stat_move(Stat& a, float m) {          // a's sums about the larger maximum m
    const float d = fmaxf((a.m - base_of(m)) * LOG2E, -200.f), f = exp2f(d);
    a.t = f * (a.t + a.s * d);
    a.s = f * a.s;
    a.m = m;
}
__device__ __forceinline__ void stat_add(Stat& a, float z) {           // z <= a.m, or NaN
    const float y = (z - base_of(a.m)) * LOG2E, e = exp2f(y);
    a.s += e;
    a.t += e * fmaxf(y, -200.f);                                       // 0 * -inf
}
__device__ __forceinline__ void stat_join(Stat& a, Stat b) {
    const float m = fmaxf(a.m, b.m);
    stat_move(a, m);
    stat_move(b, m);
    a.s += b.s;
    a.t += b.t;
}

// Order of the alternatives as one integer: larger value first, then lower index; NaN before everything, -0 as 0
__device__ __forceinline__ unsigned long long rank_of(float z, unsigned j) {
    const unsigned b = __float_as_uint(z == 0.f ? 0.f : z);
    const unsigned k = z != z ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((unsigned long long)k << 32) | (0xFFFFFFFFu - j);
}
__device__ __forceinline__ unsigned rank_index(unsigned long long r) { return 0xFFFFFFFFu - (unsigned)r; }

struct LpArgs {
    const void* z;
    const long long* target;
    long long N, L, sn, sc;
    int C, k;
    long long ignore;
    float *log_prob, *entropy, *stats, *top;
    long long* top_index;
};

// log p of the target, entropy and the saved pair of row i from its statistics
template <typename T>
__device__ __forceinline__ void lp_finish(const LpArgs& a, const T* row, long long i, const Stat& st, long long rows) {
    const float base = base_of(st.m), logs = logf(st.s);
    if (a.log_prob) {
        const long long t = a.target[i];
        float v = __builtin_nanf("");                                  // a target outside [0, C): as in the weighted cross entropy
        if (t == a.ignore) v = 0.f;
        else if (t >= 0 && t < a.C) v = (Elem<T>::ld(row + t * a.sc) - base) - logs;
        a.log_prob[i] = v;
    }
    a.entropy[i] = logs - st.t * LN2 / st.s;
    a.stats[i] = base;
    a.stats[rows + i] = logs;
}

// planes: one thread per pixel
template <typename T>
__global__ __launch_bounds__(256) void lp_planes_kernel(const LpArgs a) {
    const long long rows = a.N * a.L;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows; i += (long long)gridDim.x * 256) {
        const long long n = i / a.L, l = i % a.L;
        const T* row = (const T*)a.z + n * a.sn + l;
        Stat st{-INFINITY, 0.f, 0.f};
        for (int c = 0; c < a.C; ++c) {
            const float z = Elem<T>::ld(row + c * a.sc);
            if (z > st.m) stat_move(st, z);
            stat_add(st, z);
        }
        lp_finish(a, row, i, st, rows);
        unsigned long long last = ~0ull;
        for (int k = 0; k < a.k; ++k) {
            unsigned long long best = 0;
            for (int c = 0; c < a.C; ++c) {
                const unsigned long long r = rank_of(Elem<T>::ld(row + c * a.sc), c);
                if ((r < last || k == 0) && r > best) best = r;
            }
            last = best;
            const unsigned j = rank_index(best);
            a.top[(n * a.k + k) * a.L + l] = (Elem<T>::ld(row + j * a.sc) - base_of(st.m)) - logf(st.s);
            a.top_index[(n * a.k + k) * a.L + l] = j;
        }
    }
}

// rows: one workgroup per row
template <typename T>
__global__ __launch_bounds__(256) void lp_rows_kernel(const LpArgs a) {
    __shared__ Stat part[4];
    __shared__ unsigned long long ranks[4];
    const long long i = blockIdx.x;
    const T* row = (const T*)a.z + i * a.sn;
    Stat st{-INFINITY, 0.f, 0.f};
    for (int c = threadIdx.x; c < a.C; c += 256) {
        const float z = Elem<T>::ld(row + c);
        if (z > st.m) stat_move(st, z);
        stat_add(st, z);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) stat_join(st, Stat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)});
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = st;
    __syncthreads();
    st = part[0];
    for (int w = 1; w < 4; ++w) stat_join(st, part[w]);
    if (threadIdx.x == 0) lp_finish(a, row, i, st, a.N);
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.k; ++k) {
        unsigned long long best = 0;
        for (int c = threadIdx.x; c < a.C; c += 256) {
            const unsigned long long r = rank_of(Elem<T>::ld(row + c), c);
            if ((r < last || k == 0) && r > best) best = r;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const unsigned long long r = __shfl_xor(best, o, 64);
            best = r > best ? r : best;
        }
        __syncthreads();                                               // the previous round's ranks have been read
        if ((threadIdx.x & 63) == 0) ranks[threadIdx.x >> 6] = best;
        __syncthreads();
        for (int w = 0; w < 4; ++w) best = ranks[w] > best ? ranks[w] : best;
        last = best;
        if (threadIdx.x == 0) {
            const unsigned j = rank_index(best);
            a.top[i * a.k + k] = (Elem<T>::ld(row + j) - base_of(st.m)) - logf(st.s);
            a.top_index[i * a.k + k] = j;
        }
    }
}

struct LpBwdArgs {
    const void* z;
    const long long* target;
    long long N, L, sn, sc, dn, dc;
    int C, k;
    long long ignore;
    const float *stats, *entropy, *g_log_prob, *g_entropy, *g_top;
    const long long* top_index;
    void* dz;
};

// One element per thread; rows whose gradients are all 0 get 0 whatever their logits hold
template <typename T>
__global__ __launch_bounds__(256) void lp_bwd_kernel(const LpBwdArgs a) {
    const long long rows = a.N * a.L, total = rows * a.C;
    const bool planes = a.sc != 1;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long long)gridDim.x * 256) {
        long long n, l, c;
        if (planes) { l = e % a.L; c = e / a.L % a.C; n = e / a.L / a.C; }
        else { l = 0; c = e % a.C; n = e / a.C; }
        const long long i = n * a.L + l;
        const long long t = a.g_log_prob ? a.target[i] : a.ignore;
        const float gl = t == a.ignore ? 0.f : t >= 0 && t < a.C ? a.g_log_prob[i] : __builtin_nanf("");
        const float gh = a.g_entropy ? a.g_entropy[i] : 0.f;
        float pull = gl, own = c == t ? gl : 0.f;
        bool any = gl != 0.f || gh != 0.f;
        for (int k = 0; k < a.k && a.g_top; ++k) {
            const long long at = (n * a.k + k) * a.L + l;
            const float gk = a.g_top[at];
            any = any || gk != 0.f;
            pull += gk;
            if (a.top_index[at] == c) own += gk;
        }
        float d = 0.f;
        if (any) {
            const float lp = (Elem<T>::ld((const T*)a.z + n * a.sn + c * a.sc + l) - a.stats[i]) - a.stats[rows + i];
            const float p = exp2f(lp * LOG2E);
            d = own - p * (pull + (gh != 0.f ? gh * (fmaxf(lp, -200.f) + a.entropy[i]) : 0.f));
        }
        Elem<T>::st((T*)a.dz + n * a.dn + c * a.dc + l, d);
    }
}

static inline bool lp_shape_ok(int dtype, long long N, int C, long long L, long long sn, long long sc, int k) {
    if ((dtype != ERF_F32 && dtype != ERF_BF16) || N <= 0 || C <= 0 || L <= 0 || sn < 0 || k < 0 || k > C || k > ERF_TOP_MAX) return false;
    if (N > 0x7FFFFFFFll || L > 0x7FFFFFFFll || N * L > (1ll << 40)) return false;
    return (sc == 1 && L == 1) || (sc >= L);
}

static inline unsigned lp_grid(long long total) {
    const long long g = (total + 255) / 256;
    return (unsigned)(g > 65536 ? 65536 : g);
}

extern "C" {

int erf_class_log_probs_fwd(const void* logits, int dtype, long long N, int C, long long L, long long stride_n, long long stride_c,
                            const long long* target, long long ignore_index, float* log_prob, float* entropy, float* stats, int top_k,
                            float* top_log_probs, long long* top_indices, void* stream) {
    if (!logits || !entropy || !stats || (!target != !log_prob) || !lp_shape_ok(dtype, N, C, L, stride_n, stride_c, top_k) ||
        (top_k && (!top_log_probs || !top_indices)))
        return ERF_EINVAL;
    const LpArgs a{logits, target, N, L, stride_n, stride_c, C, top_k, ignore_index, log_prob, entropy, stats, top_log_probs, top_indices};
    hipStream_t s = (hipStream_t)stream;
    if (stride_c == 1 && L == 1) {
        if (dtype == ERF_BF16) hipLaunchKernelGGL(lp_rows_kernel<bf16raw>, dim3((unsigned)N), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(lp_rows_kernel<float>, dim3((unsigned)N), dim3(256), 0, s, a);
    } else {
        if (dtype == ERF_BF16) hipLaunchKernelGGL(lp_planes_kernel<bf16raw>, dim3(lp_grid(N * L)), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(lp_planes_kernel<float>, dim3(lp_grid(N * L)), dim3(256), 0, s, a);
    }
    return erf_check_launch();
}

int erf_class_log_probs_bwd(const void* logits, int dtype, long long N, int C, long long L, long long stride_n, long long stride_c,
                            const long long* target, long long ignore_index, const float* stats, const float* entropy,
                            const float* g_log_prob, const float* g_entropy, int top_k, const long long* top_indices, const float* g_top,
                            void* dlogits, long long dstride_n, long long dstride_c, void* stream) {
    if (!logits || !stats || !entropy || !dlogits || (g_log_prob && !target) || !lp_shape_ok(dtype, N, C, L, stride_n, stride_c, top_k) ||
        (g_top && (!top_indices || !top_k)) || dstride_n < 0 || (dstride_c == 1) != (stride_c == 1) || (dstride_c != 1 && dstride_c < L))
        return ERF_EINVAL;
    const LpBwdArgs a{logits, target, N, L, stride_n, stride_c, dstride_n, dstride_c, C, g_top ? top_k : 0, ignore_index, stats, entropy,
                      g_log_prob, g_entropy, g_top, top_indices, dlogits};
    const unsigned g = lp_grid(N * L * C);
    if (dtype == ERF_BF16) hipLaunchKernelGGL(lp_bwd_kernel<bf16raw>, dim3(g), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(lp_bwd_kernel<float>, dim3(g), dim3(256), 0, (hipStream_t)stream, a);
    return erf_check_launch();
}

}  // extern "C"
