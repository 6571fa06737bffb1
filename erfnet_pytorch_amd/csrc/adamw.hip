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
//
// 32 bits: the memory bounds it (fp32: 28 bytes an element).  8 bits: 97 M elements in bf16 (10 bytes each) 220 us, 4.4 TB/s, memory and
// arithmetic about even.  A network's 228 small tensors (2.1 M elements): 13 us in either, one launch's latency and the tail of
// the tensors that fill no chunk.
#include "../../include/erfnet_mi355.h"
#include "common.cuh"
#include <type_traits>

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

// Mixing of 32 bits by xor-shifts and odd multipliers; these are the ones that C. Wellons, "Prospecting for Hash Functions" (2018), found
// in a search for the least bias between input and output bits
__device__ __forceinline__ unsigned mix32(unsigned h) {
    h ^= h >> 16; h *= 0x7FEB352Du;
    h ^= h >> 15; h *= 0x846CA68Bu;
    return h ^ (h >> 16);
}

// x, |x| <= 448, to the e4m3 value below or above it, up with probability (16 random bits) distance / step; the sign is dropped.
// Values from 2^-6 on have 3 mantissa bits: adding random bits below them and cutting them off is the rounding.  Below 2^-6 the
// step stays 2^-9, which is the mantissa step of x + 2^-6.
__device__ __forceinline__ float round_e4m3(float x, unsigned rnd16) {
    const float up = fabsf(x) < 0.015625f ? 0.015625f : 0.f;
    const unsigned b = (__float_as_uint(fabsf(x) + up) + (rnd16 << 4)) & 0xFFF00000u;
    return __uint_as_float(b) - up;
}

// 2^e with e the smallest exponent that brings the value with bits `most` (finite, >= 0) to 448 = 1.75 * 2^8 or below
__device__ __forceinline__ int scale_exp(unsigned most) {
    const int e = (int)(most >> 23) - 127 - 8 + ((most & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return most ? min(max(e, -126), 120) : -126;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// Largest of the 64 lanes' values, as a scalar: shifts within rows of 16 lanes, then the rows' last lanes are passed on
template <int CTRL>
__device__ __forceinline__ unsigned umax_dpp(unsigned v) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return o > v ? o : v;
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
    v = umax_dpp<0x111>(v);                                   // row_shr 1, 2, 4, 8
    v = umax_dpp<0x112>(v);
    v = umax_dpp<0x114>(v);
    v = umax_dpp<0x118>(v);
    v = umax_dpp<0x142>(v);                                   // row_bcast 15, 31
    v = umax_dpp<0x143>(v);
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// Addresses from the table are global memory: said here, the compiler forms scalar base + 32-bit offset accesses
#define GLOBAL __attribute__((address_space(1)))

// One chunk's arrays, at its first element; scales at the chunk's first scale block
template <typename T, int BITS>
struct ChunkPtrs {
    typedef typename std::conditional<BITS == 32, float, unsigned char>::type S;
    GLOBAL T* p;
    const GLOBAL T* g;
    GLOBAL S *m, *v;
    GLOBAL float *sm, *sr;
    __device__ __forceinline__ ChunkPtrs(const erf_adamw_tensor& t, long long start)
        : p((GLOBAL T*)t.param + start), g((const GLOBAL T*)t.grad + start), m((GLOBAL S*)t.exp_avg + start), v((GLOBAL S*)t.exp_avg_sq + start),
          sm((GLOBAL float*)t.exp_avg_scale + start / QB), sr((GLOBAL float*)t.root_scale + start / QB) {}
};

__device__ __forceinline__ f32x4 quad(const GLOBAL float* p) { return *(const GLOBAL f32x4*)p; }
__device__ __forceinline__ f32x4 quad(const GLOBAL bf16raw* p) {
    const i32x2 r = *(const GLOBAL i32x2*)p;
    return f32x4{__uint_as_float((unsigned)r[0] << 16), __uint_as_float((unsigned)r[0] & 0xFFFF0000u), __uint_as_float((unsigned)r[1] << 16),
                 __uint_as_float((unsigned)r[1] & 0xFFFF0000u)};
}
__device__ __forceinline__ void put_quad(GLOBAL float* p, const f32x4& v) { *(GLOBAL f32x4*)p = v; }
__device__ __forceinline__ void put_quad(GLOBAL bf16raw* p, const f32x4& v) { *(GLOBAL i32x2*)p = pack_bf16x4(v); }

// One lane's 4 elements of a scale block on their way through the update; i: their place in the chunk.
// VEC: all 4 exist and lie on vector boundaries; else the first n of them, one by one.
template <typename T, int BITS>
struct Lane4 {
    f32x4 p, g, m, v;                                         // BITS 8: m and v's codes as words, decoded by the update
    int cm, cr;

    template <bool VEC>
    __device__ __forceinline__ void load(const ChunkPtrs<T, BITS>& t, unsigned i, int n) {
        if constexpr (VEC) {
            p = quad(t.p + i);
            g = quad(t.g + i);
            if constexpr (BITS == 32) { m = quad(t.m + i); v = quad(t.v + i); }
            else { cm = *(const GLOBAL int*)(t.m + i); cr = *(const GLOBAL int*)(t.v + i); }
        } else {
            cm = cr = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = e < n;
                p[e] = in ? Elem<T>::to_f32(t.p[i + e]) : 0.f;
                g[e] = in ? Elem<T>::to_f32(t.g[i + e]) : 0.f;
                if constexpr (BITS == 32) {
                    m[e] = in ? t.m[i + e] : 0.f;
                    v[e] = in ? t.v[i + e] : 0.f;
                } else if (in) {
                    cm |= t.m[i + e] << (8 * e);
                    cr |= t.v[i + e] << (8 * e);
                }
            }
        }
    }

    template <bool VEC>
    __device__ __forceinline__ void store(const ChunkPtrs<T, BITS>& t, unsigned i, int n) const {
        if constexpr (VEC) {
            put_quad(t.p + i, p);
            if constexpr (BITS == 32) { put_quad(t.m + i, m); put_quad(t.v + i, v); }
            else { *(GLOBAL int*)(t.m + i) = cm; *(GLOBAL int*)(t.v + i) = cr; }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e >= n) break;
                t.p[i + e] = Elem<T>::from_f32(p[e]);
                if constexpr (BITS == 32) { t.m[i + e] = m[e]; t.v[i + e] = v[e]; }
                else { t.m[i + e] = (unsigned char)(cm >> (8 * e)); t.v[i + e] = (unsigned char)(cr >> (8 * e)); }
            }
        }
    }
};

// plain_div: eps is not in fast_div's range (sqrt(v) / sqrt(1 - b2^t) stays below 2^120)
struct AdamwScalars { float step_size, decay, inv_bc2, b1, omb1, b2, omb2, eps; unsigned key; bool plain_div; };

// sqrt(v), v >= 0, to half a step but for one case in a million: y = v / sqrt(v) from the hardware's reciprocal root, then
// y + (v - y^2) / (2 sqrt(v)).  For 0 and normal v: the hardware's reciprocal root does not take subnormal ones.
__device__ __forceinline__ float fast_sqrt(float v) {
    const float s = __builtin_amdgcn_rsqf(fmaxf(v, 1.17549435e-38f)), y = v * s;
    return fmaf(fmaf(-y, y, v), 0.5f * s, y);
}
// m / d in the same way, for 2^-126 <= d <= 2^125: outside that 1 / d has no digits, or is infinite.  |m / d| is finite there: m came
// from gradients of which sqrt(v), in d, has its share
__device__ __forceinline__ float fast_div(float m, float d) {
    const float r = __builtin_amdgcn_rcpf(d), q = m * r;
    return fmaf(fmaf(-q, d, m), r, q);
}

// The update with moments in 32 bits.  Multiplications and additions round one by one (no fused ones), so that a plain program
// gives the same bits.
template <typename T>
__device__ __forceinline__ void adamw_update(Lane4<T, 32>& x, const AdamwScalars& k, unsigned, float&, float&) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x.m[e] = x.m[e] * k.b1 + x.g[e] * k.omb1;
        x.v[e] = x.v[e] * k.b2 + x.g[e] * x.g[e] * k.omb2;
        x.p[e] = x.p[e] * k.decay - x.m[e] / (sqrtf(x.v[e]) * k.inv_bc2 + k.eps) * k.step_size;
    }
}

// ... in 8 bits, of one wave's scale block; sm, sr: its scales, replaced by the new ones.  The arithmetic, not the memory, bounds
// this kernel: what handles values that are not finite, or v that are subnormal, stands in a branch of its own that a wave takes when
// it has met one.  Bits of NaN and infinity, as integers, are above all others, so the maximum finds them; subnormal v take a class
// compare each (97 M elements 220 us, 217 without).
template <typename T>
__device__ __forceinline__ void adamw_update(Lane4<T, 8>& x, const AdamwScalars& k, unsigned counter, float& sm, float& sr) {
#pragma clang fp contract(off)
    const f32x2 m0 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cm, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cm, true);
    const f32x2 r0 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cr, false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8(x.cr, true);
    float m[4] = {m0[0], m0[1], m1[0], m1[1]}, r[4] = {r0[0], r0[1], r1[0], r1[1]}, v[4];
    unsigned bm[4], br[4];
    bool subnormal = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float old = r[e] * sr;
        m[e] = m[e] * sm * k.b1 + x.g[e] * k.omb1;
        v[e] = old * old * k.b2 + x.g[e] * x.g[e] * k.omb2;
        r[e] = fast_sqrt(v[e]);
        bm[e] = __float_as_uint(m[e]) & 0x7FFFFFFFu;
        br[e] = __float_as_uint(r[e]);
        subnormal |= __builtin_amdgcn_classf(v[e], 0x80);     // above 0
    }
    unsigned most_m = wave_umax(max(max(bm[0], bm[1]), max(bm[2], bm[3]))), most_r = wave_umax(max(max(br[0], br[1]), max(br[2], br[3])));
    const bool odd = most_m >= 0x7F800000u || most_r >= 0x7F800000u || k.plain_div || __any(subnormal);
    if (!odd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x.p[e] = x.p[e] * k.decay - fast_div(m[e], r[e] * k.inv_bc2 + k.eps) * k.step_size;
    } else {
        // a value that is not finite becomes a NaN code and leaves its neighbours' scale alone
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            r[e] = sqrtf(v[e]);
            x.p[e] = x.p[e] * k.decay - m[e] / (r[e] * k.inv_bc2 + k.eps) * k.step_size;
            br[e] = __float_as_uint(r[e]) < 0x7F800000u ? __float_as_uint(r[e]) : 0u;
            bm[e] = bm[e] < 0x7F800000u ? bm[e] : 0u;
        }
        most_m = wave_umax(max(max(bm[0], bm[1]), max(bm[2], bm[3])));
        most_r = wave_umax(max(max(br[0], br[1]), max(br[2], br[3])));
    }
    const int em = scale_exp(most_m), er = scale_exp(most_r);
    const float im = exp2i(-em), ir = exp2i(-er);
    sm = exp2i(em);
    sr = exp2i(er);
    float qm[4], qr[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned h = mix32((counter + e) ^ k.key);
        const float tm = m[e] * im, tr = r[e] * ir;
        qm[e] = copysignf(round_e4m3(tm, h & 0xFFFFu), tm);
        qr[e] = tr > 0.f ? fmaxf(round_e4m3(tr, h >> 16), 0.001953125f) : 0.f;        // above 0 stays above 0
    }
    if (odd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            qm[e] = fabsf(m[e]) < INFINITY ? qm[e] : __builtin_nanf("");
            qr[e] = r[e] < INFINITY ? qr[e] : __builtin_nanf("");
        }
    }
    x.cm = __builtin_amdgcn_cvt_pk_fp8_f32(qm[2], qm[3], __builtin_amdgcn_cvt_pk_fp8_f32(qm[0], qm[1], 0, false), true);
    x.cr = __builtin_amdgcn_cvt_pk_fp8_f32(qr[2], qr[3], __builtin_amdgcn_cvt_pk_fp8_f32(qr[0], qr[1], 0, false), true);
}

// A workgroup takes one chunk; a wave takes every 4th scale block of it, 4 neighbouring elements per lane (16-byte accesses on
// fp32, 8 on bf16, 4 on codes).  A whole chunk on vector boundaries has all its loads in flight before the first update; what is
// ragged or lies off the boundaries goes block by block, element by element.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwArgs a) {
    constexpr int PER_WAVE = CHUNK / QB / 4;
    const int2 ch = a.chunks[blockIdx.x];
    const erf_adamw_tensor t = a.table[ch.x];
    if (!t.grad) return;                                      // the whole workgroup: no gradient, no step of this tensor
    const int step = a.steps[blockIdx.x] + 1;
    const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long start = (long long)ch.y * CHUNK;
    const ChunkPtrs<T, BITS> ptr(t, start);
    constexpr unsigned long long VT = sizeof(T) * 4 - 1, VS = BITS == 32 ? 15 : 3;
    const bool whole = start + CHUNK <= t.count && (((unsigned long long)t.param | (unsigned long long)t.grad) & VT) == 0 &&
                       (((unsigned long long)t.exp_avg | (unsigned long long)t.exp_avg_sq) & VS) == 0;
    Lane4<T, BITS> x[PER_WAVE];
    float sm[PER_WAVE], sr[PER_WAVE];
    if (whole) {
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const unsigned q = j * 4 + wave;
            x[j].template load<true>(ptr, q * QB + lane * 4, 4);
            if (BITS == 8) { sm[j] = ptr.sm[q]; sr[j] = ptr.sr[q]; }
        }
    }
    __syncthreads();                                          // every wave has read the count
    if (threadIdx.x == 0) a.steps[blockIdx.x] = step;
    const double lr = *a.lr;
    const AdamwScalars k{(float)(lr / (1.0 - ipow(a.b1, step))), (float)(1.0 - lr * a.wd), (float)(1.0 / sqrt(1.0 - ipow(a.b2, step))),
                         (float)a.b1, (float)(1.0 - a.b1), (float)a.b2, (float)(1.0 - a.b2), (float)a.eps,
                         ((unsigned)step * 0x9E3779B9u) ^ a.seed, !(a.eps >= 0x1p-126 && a.eps <= 0x1p100)};
    const unsigned counter = (unsigned)(t.base + start);
    if (whole) {
#pragma unroll
        for (int j = 0; j < PER_WAVE; ++j) {
            const unsigned q = j * 4 + wave, i = q * QB + lane * 4;
            adamw_update<T>(x[j], k, counter + i, sm[j], sr[j]);
            x[j].template store<true>(ptr, i, 4);
            if (BITS == 8 && lane == 0) { ptr.sm[q] = sm[j]; ptr.sr[q] = sr[j]; }
        }
        return;
    }
    const int count = (int)(t.count - start < CHUNK ? t.count - start : CHUNK);
    for (unsigned q = wave; q < CHUNK / QB; q += 4) {
        if ((int)(q * QB) >= count) break;                    // uniform over the wave
        const unsigned i = q * QB + lane * 4;
        const int n = min(max(count - (int)i, 0), 4);
        Lane4<T, BITS> y;
        float ym = 0.f, yr = 0.f;
        y.template load<false>(ptr, i, n);
        if (BITS == 8) { ym = ptr.sm[q]; yr = ptr.sr[q]; }
        adamw_update<T>(y, k, counter + i, ym, yr);
        y.template store<false>(ptr, i, n);
        if (BITS == 8 && lane == 0) { ptr.sm[q] = ym; ptr.sr[q] = yr; }
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
        for (int k = 0; k < n; ++k) a.g[k] = grads[i + k];
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
