// AdamW over many tensors in one launch, with the two moments in 32 or in 8 bits.
//
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A table in device memory holds one record per tensor, a second one the tensors' chunks of CHUNK elements; a workgroup takes
// one chunk.  Each chunk keeps its own step count t: its workgroup is the only reader and writer, so one launch moves the
// counts on with no second kernel and no atomics, and a captured launch counts when it is replayed.
//
// 8-bit states: m and sqrt(v) as e4m3 codes, one power of two per QB elements as scale.  A power of two costs no rounding of
// its own, and decoding is exact.  Codes are rounded up or down at random, in proportion to the distance: b2 = 0.999 moves v
// by 0.1 % a step and half an e4m3 step is 3 % to 6 %, so rounding to nearest would never let v fall.  sqrt(v) > 0 never
// becomes 0 (its smallest code stands in): the next update divides by it.  The update of p uses the new moments before they
// are rounded.
#include "../../include/erfnet_mi355.h"
#include "common.cuh"

#define CHUNK 4096
#define QB 256

static_assert(sizeof(erf_adamw_tensor) == 64, "table record");

struct AdamwArgs {
    const erf_adamw_tensor* table;
    const int2* chunks;                // (tensor, chunk of that tensor)
    int* steps;
    const double* lr;
    double b1, b2, eps, wd;
    unsigned seed;
};

// b^t by squaring: at most 2 log2(t) roundings of 2^-53
__device__ __forceinline__ double ipow(double b, int t) {
    double r = 1.0;
    for (; t; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

// The 32-bit mixing function "lowbias32" of C. Wellons' hash prospector (public domain)
__device__ __forceinline__ unsigned mix32(unsigned h) {
    h ^= h >> 16; h *= 0x7FEB352Du;
    h ^= h >> 15; h *= 0x846CA68Bu;
    return h ^ (h >> 16);
}

// x, |x| <= 448, to the e4m3 value below or above it, up with probability (16 random bits) distance / step.
// Values from 2^-6 on have 3 mantissa bits: adding random bits below them and cutting them off is the rounding.  Below 2^-6 the
// step stays 2^-9, which is the mantissa step of x + 2^-6.  least: what is above 0 stays above 0.
__device__ __forceinline__ float round_e4m3(float x, unsigned rnd16, bool least) {
    float a = fabsf(x);
    const bool low = a < 0.015625f;
    a = low ? a + 0.015625f : a;
    a = __uint_as_float((__float_as_uint(a) + (rnd16 << 4)) & 0xFFF00000u);
    a = low ? a - 0.015625f : a;
    if (least) a = x > 0.f ? fmaxf(a, 0.001953125f) : a;
    return fabsf(x) <= 448.f ? copysignf(a, x) : __builtin_nanf("");
}

// 2^e with e the smallest exponent that brings `most` to 448 = 1.75 * 2^8 or below
__device__ __forceinline__ int scale_exp(float most) {
    const unsigned b = __float_as_uint(most);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return most > 0.f ? min(max(e, -126), 120) : -126;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

template <typename T, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwArgs a) {
#pragma clang fp contract(off)
    const int2 ch = a.chunks[blockIdx.x];
    const erf_adamw_tensor t = a.table[ch.x];
    const int step = a.steps[blockIdx.x] + 1;
    __syncthreads();                                          // every wave has read the count
    if (threadIdx.x == 0) a.steps[blockIdx.x] = step;
    const double lr = *a.lr;
    const float step_size = (float)(lr / (1.0 - ipow(a.b1, step))), decay = (float)(1.0 - lr * a.wd);
    const float inv_bc2 = (float)(1.0 / sqrt(1.0 - ipow(a.b2, step)));
    const float b1 = (float)a.b1, omb1 = (float)(1.0 - a.b1), b2 = (float)a.b2, omb2 = (float)(1.0 - a.b2), eps = (float)a.eps;
    const unsigned key = ((unsigned)step * 0x9E3779B9u) ^ a.seed;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    T* p = (T*)t.param;
    const T* g = (const T*)t.grad;
    for (int q = wave; q < CHUNK / QB; q += 4) {
        const long long first = (long long)ch.y * CHUNK + q * QB, base = first + lane * 4;
        if (first >= t.count) break;                          // uniform over the wave
        float m[4], r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const long long i = base + e;
            const bool in = i < t.count;
            const float gi = in ? Elem<T>::ld(g + i) : 0.f;
            float mi, vi;
            if (BITS == 32) {
                mi = in ? ((const float*)t.exp_avg)[i] : 0.f;
                vi = in ? ((const float*)t.exp_avg_sq)[i] : 0.f;
            } else {
                const int cm = in ? ((const unsigned char*)t.exp_avg)[i] : 0, cr = in ? ((const unsigned char*)t.exp_avg_sq)[i] : 0;
                mi = __builtin_amdgcn_cvt_f32_fp8(cm, 0) * t.exp_avg_scale[first / QB];
                vi = __builtin_amdgcn_cvt_f32_fp8(cr, 0) * t.root_scale[first / QB];
                vi = vi * vi;
            }
            mi = mi * b1 + gi * omb1;
            vi = vi * b2 + gi * gi * omb2;
            const float ri = sqrtf(vi);
            if (in) {
                Elem<T>::st(p + i, Elem<T>::ld(p + i) * decay - mi / (ri * inv_bc2 + eps) * step_size);
                if (BITS == 32) { ((float*)t.exp_avg)[i] = mi; ((float*)t.exp_avg_sq)[i] = vi; }
            }
            m[e] = mi; r[e] = ri;
        }
        if (BITS == 8) {
            // a value that is not finite becomes a NaN code and leaves its neighbours' scale alone
            float am = 0.f, ar = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                am = fmaxf(am, fabsf(m[e]) < INFINITY ? fabsf(m[e]) : 0.f);
                ar = fmaxf(ar, r[e] < INFINITY ? r[e] : 0.f);
            }
            const int em = scale_exp(wave_max(am)), er = scale_exp(wave_max(ar));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const long long i = base + e;
                if (i >= t.count) break;
                const unsigned h = mix32((unsigned)(t.base + i) ^ key);
                const float qm = round_e4m3(m[e] * exp2i(-em), h & 0xFFFFu, false), qr = round_e4m3(r[e] * exp2i(-er), h >> 16, true);
                ((unsigned char*)t.exp_avg)[i] = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(qm, qm, 0, false);
                ((unsigned char*)t.exp_avg_sq)[i] = (unsigned char)__builtin_amdgcn_cvt_pk_fp8_f32(qr, qr, 0, false);
            }
            if (lane == 0) { t.exp_avg_scale[first / QB] = exp2i(em); t.root_scale[first / QB] = exp2i(er); }
        }
    }
}

// Gradients are new tensors at new addresses after every zero_grad(set_to_none=True).  Their addresses travel as kernel
// arguments: no host buffer has to outlive the call, and a captured launch replays its own.
#define GRADS_PER_LAUNCH 256
struct AdamwGrads { const void* g[GRADS_PER_LAUNCH]; };

__global__ void adamw_grads_kernel(erf_adamw_tensor* table, int count, const AdamwGrads a) {
    const int i = threadIdx.x;
    if (i < count) table[i].grad = a.g[i];
}

extern "C" {

int erf_adamw_chunk_elements(void) { return CHUNK; }
int erf_adamw_scale_block(void) { return QB; }

int erf_adamw_set_grads(erf_adamw_tensor* table, const void* const* grads, int count, void* stream) {
    if (!table || !grads || count <= 0) return ERF_EINVAL;
    for (int i = 0; i < count; i += GRADS_PER_LAUNCH) {
        const int n = count - i < GRADS_PER_LAUNCH ? count - i : GRADS_PER_LAUNCH;
        AdamwGrads a = {};
        for (int k = 0; k < n; ++k) {
            if (!grads[i + k]) return ERF_EINVAL;
            a.g[k] = grads[i + k];
        }
        hipLaunchKernelGGL(adamw_grads_kernel, dim3(1), dim3(GRADS_PER_LAUNCH), 0, (hipStream_t)stream, table + i, n, a);
    }
    return erf_check_launch();
}

int erf_adamw_step(const erf_adamw_tensor* table, const int* chunks, int* steps, int n_chunks, const double* lr, double beta1,
                   double beta2, double eps, double weight_decay, int dtype, int state_bits, unsigned seed, void* stream) {
    if (!table || !chunks || !steps || !lr || n_chunks <= 0 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) ||
        !(eps >= 0) || (state_bits != 32 && state_bits != 8) || (dtype != ERF_F32 && dtype != ERF_BF16))
        return ERF_EINVAL;
    const AdamwArgs a{table, (const int2*)chunks, steps, lr, beta1, beta2, eps, weight_decay, seed};
    const dim3 grid((unsigned)n_chunks), block(256);
    if (dtype == ERF_F32 && state_bits == 32) hipLaunchKernelGGL((adamw_kernel<float, 32>), grid, block, 0, (hipStream_t)stream, a);
    else if (dtype == ERF_F32) hipLaunchKernelGGL((adamw_kernel<float, 8>), grid, block, 0, (hipStream_t)stream, a);
    else if (state_bits == 32) hipLaunchKernelGGL((adamw_kernel<bf16raw, 32>), grid, block, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((adamw_kernel<bf16raw, 8>), grid, block, 0, (hipStream_t)stream, a);
    return erf_check_launch();
}

}  // extern "C"
