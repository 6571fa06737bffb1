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

template <typename T> struct Quad;                            // 4 neighbouring values in memory
template <> struct Quad<float> { typedef f32x4 raw; };
template <> struct Quad<bf16raw> { typedef i32x2 raw; };

// One lane's 4 elements of a scale block on their way through the update
template <typename T, int BITS>
struct Lane4 {
    f32x4 p, g, m, v;                                         // BITS 8: m and v's codes as words, decoded by update()
    int cm, cr;

    // VEC: all 4 elements exist and lie on vector boundaries; else n of them, one by one
    template <bool VEC>
    __device__ __forceinline__ void load(const erf_adamw_tensor& t, long long i, int n) {
        if (VEC) {
            p = load4((const T*)t.param + i);
            g = load4((const T*)t.grad + i);
            if (BITS == 32) { m = *(const f32x4*)((const float*)t.exp_avg + i); v = *(const f32x4*)((const float*)t.exp_avg_sq + i); }
            else { cm = *(const int*)((const char*)t.exp_avg + i); cr = *(const int*)((const char*)t.exp_avg_sq + i); }
            return;
        }
        cm = cr = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = e < n;
            p[e] = in ? Elem<T>::ld((const T*)t.param + i + e) : 0.f;
            g[e] = in ? Elem<T>::ld((const T*)t.grad + i + e) : 0.f;
            if (BITS == 32) {
                m[e] = in ? ((const float*)t.exp_avg)[i + e] : 0.f;
                v[e] = in ? ((const float*)t.exp_avg_sq)[i + e] : 0.f;
            } else if (in) {
                cm |= ((const unsigned char*)t.exp_avg)[i + e] << (8 * e);
                cr |= ((const unsigned char*)t.exp_avg_sq)[i + e] << (8 * e);
            }
        }
    }

    template <bool VEC>
    __device__ __forceinline__ void store(const erf_adamw_tensor& t, long long i, int n) const {
        if (VEC) {
            store4((T*)t.param + i, p);
            if (BITS == 32) { *(f32x4*)((float*)t.exp_avg + i) = m; *(f32x4*)((float*)t.exp_avg_sq + i) = v; }
            else { *(int*)((char*)t.exp_avg + i) = cm; *(int*)((char*)t.exp_avg_sq + i) = cr; }
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e >= n) break;
            Elem<T>::st((T*)t.param + i + e, p[e]);
            if (BITS == 32) { ((float*)t.exp_avg)[i + e] = m[e]; ((float*)t.exp_avg_sq)[i + e] = v[e]; }
            else { ((unsigned char*)t.exp_avg)[i + e] = cm >> (8 * e); ((unsigned char*)t.exp_avg_sq)[i + e] = cr >> (8 * e); }
        }
    }
};

struct AdamwScalars { float step_size, decay, inv_bc2, b1, omb1, b2, omb2, eps; unsigned key; };

// The update of one wave's scale block, QB elements from `first` on; sm, sr: its scales, replaced by the new ones
template <typename T, int BITS>
__device__ __forceinline__ void adamw_update(Lane4<T, BITS>& x, const AdamwScalars& k, unsigned counter, float& sm, float& sr) {
#pragma clang fp contract(off)
    if (BITS == 8) {
        const f32x2 m0 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cm, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cm, true);
        const f32x2 r0 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cr, false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cr, true);
        x.m = f32x4{m0[0], m0[1], m1[0], m1[1]};
        x.v = f32x4{r0[0], r0[1], r1[0], r1[1]};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float r = x.v[e] * sr;
            x.m[e] *= sm;
            x.v[e] = r * r;
        }
    }
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x.m[e] = x.m[e] * k.b1 + x.g[e] * k.omb1;
        x.v[e] = x.v[e] * k.b2 + x.g[e] * x.g[e] * k.omb2;
        r[e] = sqrtf(x.v[e]);
        x.p[e] = x.p[e] * k.decay - x.m[e] / (r[e] * k.inv_bc2 + k.eps) * k.step_size;
    }
    if (BITS == 8) {
        // a value that is not finite becomes a NaN code and leaves its neighbours' scale alone
        float am = 0.f, ar = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            am = fmaxf(am, fabsf(x.m[e]) < INFINITY ? fabsf(x.m[e]) : 0.f);
            ar = fmaxf(ar, r[e] < INFINITY ? r[e] : 0.f);
        }
        const int em = scale_exp(wave_max(am)), er = scale_exp(wave_max(ar));
        const float im = exp2i(-em), ir = exp2i(-er);
        sm = exp2i(em);
        sr = exp2i(er);
        float qm[4], qr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned h = mix32((counter + e) ^ k.key);
            qm[e] = round_e4m3(x.m[e] * im, h & 0xFFFFu, false);
            qr[e] = round_e4m3(r[e] * ir, h >> 16, true);
        }
        x.cm = __builtin_amdgcn_cvt_pk_fp8_f32(qm[2], qm[3], __builtin_amdgcn_cvt_pk_fp8_f32(qm[0], qm[1], 0, false), true);
        x.cr = __builtin_amdgcn_cvt_pk_fp8_f32(qr[2], qr[3], __builtin_amdgcn_cvt_pk_fp8_f32(qr[0], qr[1], 0, false), true);
    }
}

// A workgroup takes one chunk; a wave takes every 4th scale block of it, 4 neighbouring elements per lane (16-byte accesses on
// fp32, 8 on bf16, 4 on codes).  A whole chunk on vector boundaries has all its loads in flight before the first update; what is
// ragged or lies off the boundaries goes block by block, element by element.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwArgs a) {
    constexpr int PER_WAVE = CHUNK / QB / 4;
    const int2 ch = a.chunks[blockIdx.x];
    const erf_adamw_tensor t = a.table[ch.x];
    const int step = a.steps[blockIdx.x] + 1;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long start = (long long)ch.y * CHUNK;
    const unsigned long long at = (unsigned long long)t.param | (unsigned long long)t.grad |
                                  (BITS == 32 ? (unsigned long long)t.exp_avg | (unsigned long long)t.exp_avg_sq : 0ull);
    const bool whole = start + CHUNK <= t.count && at % sizeof(typename Quad<T>::raw) == 0 &&
                       (BITS == 8 ? ((unsigned long long)t.exp_avg | (unsigned long long)t.exp_avg_sq) % 4 == 0
                                  : ((unsigned long long)t.exp_avg | (unsigned long long)t.exp_avg_sq) % 16 == 0);
    Lane4<T, BITS> x[PER_WAVE];
    float sm[PER_WAVE], sr[PER_WAVE];
    if (whole) {
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const int q = j * 4 + wave;
            x[j].template load<true>(t, start + q * QB + lane * 4, 4);
            if (BITS == 8) { sm[j] = t.exp_avg_scale[start / QB + q]; sr[j] = t.root_scale[start / QB + q]; }
        }
    }
    __syncthreads();                                          // every wave has read the count
    if (threadIdx.x == 0) a.steps[blockIdx.x] = step;
    const double lr = *a.lr;
    const AdamwScalars k{(float)(lr / (1.0 - ipow(a.b1, step))), (float)(1.0 - lr * a.wd), (float)(1.0 / sqrt(1.0 - ipow(a.b2, step))),
                         (float)a.b1, (float)(1.0 - a.b1), (float)a.b2, (float)(1.0 - a.b2), (float)a.eps,
                         ((unsigned)step * 0x9E3779B9u) ^ a.seed};
    if (whole) {
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const int q = j * 4 + wave;
            const long long i = start + q * QB + lane * 4;
            adamw_update<T, BITS>(x[j], k, (unsigned)(t.base + i), sm[j], sr[j]);
            x[j].template store<true>(t, i, 4);
            if (BITS == 8 && lane == 0) { t.exp_avg_scale[start / QB + q] = sm[j]; t.root_scale[start / QB + q] = sr[j]; }
        }
        return;
    }
    for (int q = wave; q < CHUNK / QB; q += 4) {
        const long long first = start + q * QB, i = first + lane * 4;
        if (first >= t.count) break;                          // uniform over the wave
        const long long left = t.count - i;
        const int n = left > 4 ? 4 : left < 0 ? 0 : (int)left;
        Lane4<T, BITS> y;
        float ym = 0.f, yr = 0.f;
        y.template load<false>(t, i, n);
        if (BITS == 8) { ym = t.exp_avg_scale[first / QB]; yr = t.root_scale[first / QB]; }
        adamw_update<T, BITS>(y, k, (unsigned)(t.base + i), ym, yr);
        y.template store<false>(t, i, n);
        if (BITS == 8 && lane == 0) { t.exp_avg_scale[first / QB] = ym; t.root_scale[first / QB] = yr; }
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
