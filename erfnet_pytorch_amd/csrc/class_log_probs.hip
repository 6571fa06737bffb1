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
    const float d = fmaxf((a.m - base_of(m)) * LOG2E, -200.f), f = __builtin_amdgcn_exp2f(d);
    a.t = f * (a.t + a.s * d);
    a.s = f * a.s;
    a.m = m;
}
__device__ __forceinline__ void stat_add(Stat& a, float base, float z) {          // base = base_of(a.m), z <= a.m or NaN
    const float y = (z - base) * LOG2E, e = __builtin_amdgcn_exp2f(y);
    a.s += e;
    a.t += e * fmaxf(y, -200.f);                                       // 0 * -inf; NaN comes through e
}
// The largest of N values, two to an instruction; NaN if one is, which leaves the running maximum as it is: the sums are NaN then
template <int N, typename VALUE>
__device__ __forceinline__ float largest(VALUE value) {
    float m = value(0);
#pragma unroll
    for (int i = 1; i < N; ++i) m = __builtin_elementwise_maximum(m, value(i));
    return m;
}

// Order of the alternatives as one integer: larger value first, then lower index; NaN before everything, -0 as 0.  No rank
// is 0 or ~0: these stand for nothing and for a bound above all.
typedef unsigned long long u64;
__device__ __forceinline__ u64 rank_of(float z, unsigned j) {
    const unsigned b = __float_as_uint(z == 0.f ? 0.f : z);
    const unsigned k = z != z ? 0xFFFFFFFEu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((u64)k << 32) | (0xFFFFFFFFu - j);
}
__device__ __forceinline__ unsigned rank_index(u64 r) { return 0xFFFFFFFFu - (unsigned)r; }
__device__ __forceinline__ float rank_value(u64 r) {
    const unsigned k = (unsigned)(r >> 32);
    return k > 0xFF800000u ? __builtin_nanf("") : __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

// Reductions over teams of 8, 16 or 64 lanes; every lane of the team gets the result.  8 and 16 lanes: exchanges within a row of 16
// (across 1, 2 and 4 lanes, then 8); 64: shifts within rows, then the rows' last lanes are passed on and lane 63 has the result.
// Lanes without a partner read 0, which is below every rank and adds nothing.
template <int CTRL> __device__ __forceinline__ int dpp0(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true); }
template <int CTRL> __device__ __forceinline__ float dpp_f(float v) { return __int_as_float(dpp0<CTRL>(__float_as_int(v))); }
template <int CTRL> __device__ __forceinline__ u64 dpp_u(u64 v) {
    return ((u64)(unsigned)dpp0<CTRL>((int)(v >> 32)) << 32) | (unsigned)dpp0<CTRL>((int)v);
}
#define SWAP1 0xB1       // quad_perm 1,0,3,2
#define SWAP2 0x4E       // quad_perm 2,3,0,1
#define MIRROR8 0x141    // row_half_mirror: after the first two, lane and mirror image stand for the two quads
#define ROTATE8 0x128    // row_ror 8
template <int TEAM> __device__ __forceinline__ float team_sum(float v) {
    if (TEAM == 64) {
        v += dpp_f<0x111>(v); v += dpp_f<0x112>(v); v += dpp_f<0x114>(v); v += dpp_f<0x118>(v); v += dpp_f<0x142>(v); v += dpp_f<0x143>(v);
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
    }
    v += dpp_f<SWAP1>(v); v += dpp_f<SWAP2>(v); v += dpp_f<MIRROR8>(v);
    if (TEAM == 16) v += dpp_f<ROTATE8>(v);
    return v;
}
template <int TEAM> __device__ __forceinline__ u64 team_best(u64 v) {
    auto up = [&](u64 o) { v = o > v ? o : v; };
    if (TEAM == 64) {
        up(dpp_u<0x111>(v)); up(dpp_u<0x112>(v)); up(dpp_u<0x114>(v)); up(dpp_u<0x118>(v)); up(dpp_u<0x142>(v)); up(dpp_u<0x143>(v));
        return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, 63);
    }
    up(dpp_u<SWAP1>(v)); up(dpp_u<SWAP2>(v)); up(dpp_u<MIRROR8>(v));
    if (TEAM == 16) up(dpp_u<ROTATE8>(v));
    return v;
}
template <int CTRL> __device__ __forceinline__ float dpp_largest(float v) {           // lanes without a partner keep their own
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, 0xF, 0xF, false)));
}
template <int TEAM> __device__ __forceinline__ float team_largest(float v) {
    if (TEAM == 64) {
        v = dpp_largest<0x111>(v); v = dpp_largest<0x112>(v); v = dpp_largest<0x114>(v); v = dpp_largest<0x118>(v);
        v = dpp_largest<0x142>(v); v = dpp_largest<0x143>(v);
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
    }
    v = fmaxf(v, dpp_f<SWAP1>(v)); v = fmaxf(v, dpp_f<SWAP2>(v)); v = fmaxf(v, dpp_f<MIRROR8>(v));
    if (TEAM == 16) v = fmaxf(v, dpp_f<ROTATE8>(v));
    return v;
}

struct LpArgs {
    const void* z;
    const long long* target;
    long long N, L, sn, sc;
    int C, k;
    long long ignore;
    float *log_prob, *entropy, *stats, *top;
    long long* top_index;
    int segments;                      // rows: workgroups per row
    long long first;                   // rows: the launch's first one
    u64* parts;                        // [N][segments][2 + k]: (m, s), (t, -), the segment's best ranks
};

// The target's logit of row i, fetched while the row is on its way; NaN for a target outside [0, C), as in the weighted cross entropy
struct LpTarget { float z; bool ignored; };
template <typename T>
__device__ __forceinline__ LpTarget lp_target(const LpArgs& a, const T* row, long long i) {
    LpTarget q{__builtin_nanf(""), false};
    if (a.log_prob) {
        const long long t = a.target[i];
        q.ignored = t == a.ignore;
        if (t >= 0 && t < a.C) q.z = Elem<T>::ld(row + t);
    }
    return q;
}
// log p of the target, entropy and the saved pair of row i from its statistics
__device__ __forceinline__ void lp_finish(const LpArgs& a, const LpTarget& q, long long i, const Stat& st, float logs) {
    const float base = base_of(st.m);
    if (a.log_prob) a.log_prob[i] = q.ignored ? 0.f : (q.z - base) - logs;
    a.entropy[i] = logs - st.t * LN2 / st.s;
    if (a.stats) {
        a.stats[i] = base;
        a.stats[a.N * a.L + i] = logs;
    }
}

// ------------------------------------------------------------------------------------------------ one thread per position
// Planes, and rows of few classes.  A thread takes P neighbouring positions (P > 1: planes, whole vectors) and BATCH classes at a
// time, all of whose loads are in flight together and which share one change of the maximum.  Up to KT alternatives are kept in
// registers, sorted; more (KT < 0) are found by rounds over the classes, as they are where NaN or too few finite values upset the order.
// Bound by the memory on planes: 6 x 20 x 512 x 1024 fp32 65 us (5.0 TB/s), with 2 alternatives, 24 bytes a position each, 84 us (4.8).
#define BATCH 8

// P neighbouring values as they lie in memory, taken apart after all loads of a set
template <typename T, int P> struct Positions;
template <> struct Positions<float, 1> { float raw; };
template <> struct Positions<float, 4> { f32x4 raw; };
template <> struct Positions<bf16raw, 1> { bf16raw raw; };
template <> struct Positions<bf16raw, 4> { i32x2 raw; };
template <typename T, int P>
__device__ __forceinline__ Positions<T, P> read_positions(const T* p) {
    return Positions<T, P>{*(const decltype(Positions<T, P>::raw)*)p};
}
template <typename T, int P>
__device__ __forceinline__ void position_values(const Positions<T, P>& v, float* f) {
    if constexpr (P == 1) f[0] = Elem<T>::to_f32(v.raw);
    else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = v.raw[i];
    } else {
        f[0] = __uint_as_float((unsigned)v.raw[0] << 16); f[1] = __uint_as_float((unsigned)v.raw[0] & 0xFFFF0000u);
        f[2] = __uint_as_float((unsigned)v.raw[1] << 16); f[3] = __uint_as_float((unsigned)v.raw[1] & 0xFFFF0000u);
    }
}
template <typename T, int P>
__device__ __forceinline__ void load_positions(const T* p, float* f) { position_values<T, P>(read_positions<T, P>(p), f); }

template <typename T, int P>
__device__ __forceinline__ void store_positions(T* p, const float* f) {
    if constexpr (P == 1) Elem<T>::st(p, f[0]);
    else if constexpr (sizeof(T) == 4) *(f32x4*)p = f32x4{f[0], f[1], f[2], f[3]};
    else *(i32x2*)p = pack_bf16x4(f32x4{f[0], f[1], f[2], f[3]});
}

template <int P>
__device__ __forceinline__ void load_indices(const long long* p, int* t) {         // classes fit 32 bits; others become -1
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const long long v = p[i];
        t[i] = v >= 0 && v <= 0x7FFFFFFF ? (int)v : -1;
    }
}
template <int P>
__device__ __forceinline__ void store_indices(long long* p, const int* t) {
    if constexpr (P == 4) {
        *(i32x4*)p = i32x4{t[0], t[0] >> 31, t[1], t[1] >> 31};
        *(i32x4*)(p + 2) = i32x4{t[2], t[2] >> 31, t[3], t[3] >> 31};
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) p[i] = t[i];
    }
}

// image and place in the image of position i: one division, of 32 bits where that does
__device__ __forceinline__ void split_position(long long i, long long L, long long& n, long long& l) {
    if (L == 1) { n = i; l = 0; }
    else if (i <= 0xFFFFFFFFll) { n = (unsigned)i / (unsigned)L; l = i - n * L; }
    else { n = i / L; l = i - n * L; }
}

template <typename T, int P, int KT>
__global__ __launch_bounds__(256) void lp_position_kernel(const LpArgs a) {
    constexpr int K = KT > 0 ? KT : 1;
    const long long rows = a.N * a.L;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * P; i < rows; i += (long long)gridDim.x * 256 * P) {
        long long n, l;
        split_position(i, a.L, n, l);
        const T* row = (const T*)a.z + n * a.sn + l;
        Stat st[P];
        float tv[P][K], zt[P];
        int tc[P][K], t[P], ignored = 0;
        if (a.log_prob) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const long long v = a.target[i + p];
                t[p] = v >= 0 && v < a.C ? (int)v : -1;
                ignored |= (v == a.ignore) << p;
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            st[p] = Stat{-INFINITY, 0.f, 0.f};
            zt[p] = __builtin_nanf("");                                // a target outside [0, C): as in the weighted cross entropy
#pragma unroll
            for (int k = 0; k < K; ++k) { tv[p][k] = -INFINITY; tc[p][k] = -1; }
        }
        for (int c0 = 0; c0 < a.C; c0 += BATCH) {
            Positions<T, P> raw[BATCH];
            float f[BATCH][P];
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (c0 + b < a.C) raw[b] = read_positions<T, P>(row + (c0 + b) * a.sc);
#pragma unroll
            for (int b = 0; b < BATCH; ++b) {
                position_values<T, P>(raw[b], f[b]);
#pragma unroll
                for (int p = 0; p < P; ++p) f[b][p] = c0 + b < a.C ? f[b][p] : -INFINITY;
            }
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float most = largest<BATCH>([&](int b) { return f[b][p]; });
                if (most > st[p].m) stat_move(st[p], most);
                const float base = base_of(st[p].m);
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                    stat_add(st[p], base, f[b][p]);
                    if (a.log_prob) zt[p] = t[p] == c0 + b ? f[b][p] : zt[p];
                    if (KT > 0) {
                        const float z = f[b][p];
                        bool up[K];                                    // slots that are sorted behind z; equal values stay before it
#pragma unroll
                        for (int k = 0; k < K; ++k) up[k] = z > tv[p][k];
#pragma unroll
                        for (int k = K - 1; k >= 0; --k) {
                            const bool from_above = k > 0 && up[k > 0 ? k - 1 : 0];
                            tv[p][k] = from_above ? tv[p][k > 0 ? k - 1 : 0] : up[k] ? z : tv[p][k];
                            tc[p][k] = from_above ? tc[p][k > 0 ? k - 1 : 0] : up[k] ? c0 + b : tc[p][k];
                        }
                    }
                }
            }
        }
        float logs[P], base[P], v[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            logs[p] = logf(st[p].s);
            base[p] = base_of(st[p].m);
        }
        if (a.log_prob) {
#pragma unroll
            for (int p = 0; p < P; ++p) v[p] = ignored >> p & 1 ? 0.f : (zt[p] - base[p]) - logs[p];
            store_positions<float, P>(a.log_prob + i, v);
        }
#pragma unroll
        for (int p = 0; p < P; ++p) v[p] = logs[p] - st[p].t * LN2 / st[p].s;
        store_positions<float, P>(a.entropy + i, v);
        if (a.stats) {
            store_positions<float, P>(a.stats + i, base);
            store_positions<float, P>(a.stats + rows + i, logs);
        }
        if (KT == 0) continue;
        bool rounds = KT < 0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            rounds = rounds || logs[p] != logs[p];
#pragma unroll
            for (int k = 0; k < K; ++k) rounds = rounds || (k < a.k && tc[p][k] < 0);
        }
        if (!rounds) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (k < a.k) {
                    int j[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) { v[p] = (tv[p][k] - base[p]) - logs[p]; j[p] = tc[p][k]; }
                    store_positions<float, P>(a.top + (n * a.k + k) * a.L + l, v);
                    store_indices<P>(a.top_index + (n * a.k + k) * a.L + l, j);
                }
            continue;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            u64 last = ~0ull;
            for (int k = 0; k < a.k; ++k) {
                u64 best = 0;
                for (int c = 0; c < a.C; ++c) {
                    const u64 r = rank_of(Elem<T>::ld(row + p + c * a.sc), c);
                    best = r < last && r > best ? r : best;
                }
                last = best;
                a.top[(n * a.k + k) * a.L + l + p] = (rank_value(best) - base[p]) - logs[p];
                a.top_index[(n * a.k + k) * a.L + l + p] = rank_index(best);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ a team of threads per row
// A row is cut at the 16-byte boundaries of memory into chunks of EPC classes, the first and the last possibly partial; thread r of
// the team takes chunks r, r + TEAM, ...  U of them are in flight and share one change of the maximum; those behind the row's end are
// skipped by the whole wave (20000 x 2048 bf16 38 us against 59).  Teams of 8, 16 or 64 lanes have the whole row in registers then; a
// workgroup goes on along a longer row.
//
// Alternatives: the k-th largest of the threads' own maxima is a bound that the k best classes reach, and few others do.  What
// reaches it is collected -- from the registers, or by the whole workgroup from the chunks of the threads whose maximum reaches it --
// and put in its place by counting.  Rows with NaN, rows where more values tie than the collection holds, and rows masked so far that
// fewer than k threads have a finite value (all the rest tie then) go through k rounds over the row: 4096 x 32000 bf16 with 5
// alternatives 58 us, and so with 50 finite logits a row or whole numbers; with 3 finite ones, or all equal, 900.  100000 x 1000: 78
// and 770.
//
// Bound by the memory where rows are long (4096 x 32000 and x 32001 bf16 52 us, 5.0 TB/s, other logits every time; 71 to 81 right behind
// a backward pass of them, which has written as much; fp32 93 us, 5.6 TB/s), by the arithmetic where the
// logits come out of the cache (8 instructions a value, one of them an exp), and by the selection, 0.5 ns a row: 100000 x 1000 fp32
// 68 us, with 5 alternatives 123; bf16 43 and 80.  The loads of the next set ahead of the work on this one gained nothing here.

template <int TEAM> struct TeamShared {
    enum { CAND = TEAM == 256 ? 512 : TEAM == 64 ? 256 : 64 };
    float m[4], s[4], t[4];
    u64 cand[CAND];
    float max[TEAM == 256 ? 256 : 1];
    int winner[TEAM == 256 ? 256 : 1];
    int winners, ncand;
    float least;
};

template <int TEAM> __device__ __forceinline__ void team_sync() {
    if (TEAM < 256) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

// Where the logits begin and end.  A row's first and last chunk may hold classes of its neighbours: within these bounds they are read
// whole all the same (100000 x 1001 bf16 75 us against 95 where they are gathered), and what is not the row's is masked afterwards.
template <typename T> struct Span { const T *first, *last; };
template <typename T, typename ARGS>
__device__ __forceinline__ Span<T> span_of(const ARGS& a) { return Span<T>{(const T*)a.z, (const T*)a.z + (a.N - 1) * a.sn + a.C}; }

// Chunk q of a row whose first class lies `off` classes behind a boundary, as it lies in memory.
// It is taken apart by chunk_values, after all loads of a set: taken apart behind the branch, each load would be waited for alone.
template <typename T>
__device__ __forceinline__ i32x4 load_chunk(const Span<T>& span, const T* row, int off, int C, int q) {
    constexpr int E = Elem<T>::EPC;
    const int c0 = q * E - off;
    const T* p = row + c0;
    if (p >= span.first && p + E <= span.last) return *(const i32x4*)p;
    i32x4 r;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if constexpr (E == 4) {
            r[w] = c0 + w >= 0 && c0 + w < C ? __float_as_int(row[c0 + w]) : 0;
        } else {
            const int c = c0 + 2 * w;
            const unsigned lo = c >= 0 && c < C ? row[c] : 0u, hi = c + 1 >= 0 && c + 1 < C ? row[c + 1] : 0u;
            r[w] = (int)(lo | hi << 16);
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void chunk_values(const i32x4& r, float* f) {
    constexpr int E = Elem<T>::EPC;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (E == 4) f[e] = __int_as_float(r[e & 3]);
        else f[e] = (e & 1) ? __uint_as_float((unsigned)r[(e >> 1) & 3] & 0xFFFF0000u) : __uint_as_float((unsigned)r[(e >> 1) & 3] << 16);
    }
}
#define NO_CLASSES(T) (Elem<T>::EPC == 4 ? (int)0xFF800000u : (int)0xFF80FF80u)          // -inf in every place of a word
// ... with -inf for what is not the row's
template <typename T>
__device__ __forceinline__ void row_values(const i32x4& r, int off, int C, int q, float* f) {
    constexpr int E = Elem<T>::EPC;
    const int c0 = q * E - off;
    chunk_values<T>(r, f);
    if (c0 < 0 || c0 + E > C) {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = c0 + e >= 0 && c0 + e < C ? f[e] : -INFINITY;
    }
}

// How many of n ranks in LDS are above r; 8 reads are in flight together
__device__ __forceinline__ int count_above(const u64* ranks, int n, u64 r) {
    int above = 0, o = 0;
    for (; o + 8 <= n; o += 8) {
        u64 v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ranks[o + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) above += v[e] > r;
    }
    for (; o < n; ++o) above += ranks[o] > r;
    return above;
}

// Best rank below `last` among the classes of chunks [q0, q1), by the whole team
template <typename T, int TEAM>
__device__ __forceinline__ u64 team_round(TeamShared<TEAM>& sh, const T* row, int off, int C, int q0, int q1, int tid, u64 last) {
    constexpr int E = Elem<T>::EPC;
    u64 best = 0;
    const int c1 = min(q1 * E - off, C);
    for (int c = max(q0 * E - off, 0) + tid; c < c1; c += TEAM) {
        const u64 r = rank_of(Elem<T>::ld(row + c), c);
        if (r < last && r > best) best = r;
    }
    if constexpr (TEAM < 256) return team_best<TEAM>(best);
    best = team_best<64>(best);
    __syncthreads();                                                   // the previous round's ranks have been read
    if ((tid & 63) == 0) sh.cand[tid >> 6] = best;
    __syncthreads();
    best = sh.cand[0];
    for (int w = 1; w < 4; ++w) best = sh.cand[w] > best ? sh.cand[w] : best;
    return best;
}

// The k-th largest of the wave's or sub-wave team's PER values a lane; -inf where there are fewer
template <int TEAM, int PER>
__device__ __forceinline__ float kth_largest(float* v, int k, int tid) {
    float m = INFINITY;
    for (int n = 0; n < k; ++n) {
        float mine = v[0];
#pragma unroll
        for (int w = 1; w < PER; ++w) mine = fmaxf(mine, v[w]);
        m = team_largest<TEAM>(mine);
        if (m == -INFINITY) break;
        // one of the lanes that have it gives it up
        const u64 have = __ballot(mine == m) & (TEAM == 64 ? ~0ull : ((1ull << (TEAM & 63)) - 1) << ((threadIdx.x & 63) - tid));
        if ((int)(threadIdx.x & 63) == __ffsll((long long)have) - 1) {
            bool gone = false;
#pragma unroll
            for (int w = 0; w < PER; ++w) {
                const bool it = !gone && v[w] == m;
                v[w] = it ? -INFINITY : v[w];
                gone = gone || it;
            }
        }
    }
    return m;
}

template <typename T, int TEAM, int U, bool TOP>
__global__ __launch_bounds__(256, TEAM == 256 ? 7 : U == 4 ? 5 : 4) void lp_rows_kernel(const LpArgs a) {
    constexpr int E = Elem<T>::EPC;
    __shared__ TeamShared<TOP || TEAM == 256 ? TEAM : 8> shared[TOP || TEAM == 256 ? 256 / TEAM : 1];
    const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM;
    const long long i = a.first + (long long)blockIdx.x * (256 / TEAM) + team;
    if (TEAM < 256 && i >= a.N) return;                                // no barrier of the workgroup below for teams within a wave
    auto& sh = shared[TOP ? team : 0];
    const T* row = (const T*)a.z + i * a.sn;
    const int off = (int)(((unsigned long long)row / sizeof(T)) % E);
    const int chunks = (a.C + off + E - 1) / E, per = (chunks + a.segments - 1) / a.segments;
    const int seg = blockIdx.y, q0 = min(seg * per, chunks), q1 = min(q0 + per, chunks);

    const Span<T> span = span_of<T>(a);
    LpTarget target{};
    if (tid == 0 && a.segments == 1) target = lp_target(a, row, i);
    Stat st{-INFINITY, 0.f, 0.f};
    float f[U][E];
    const int end = TEAM < 256 ? (a.C + 2 * (E - 1)) / E : q1;                // the chunks of any row: one bound for the whole wave
    for (int q = q0; q < (TEAM < 256 ? 1 : q1); q += TEAM * U) {
        i32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u] = i32x4{NO_CLASSES(T), NO_CLASSES(T), NO_CLASSES(T), NO_CLASSES(T)};
            if (q + u * TEAM + tid < q1) raw[u] = load_chunk(span, row, off, a.C, q + u * TEAM + tid);
        }
        float most = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + u * TEAM < end) {
                row_values<T>(raw[u], off, a.C, q + u * TEAM + tid, f[u]);
                most = __builtin_elementwise_maximum(most, largest<E>([&](int e) { return f[u][e]; }));
            }
        if (most > st.m) stat_move(st, most);
        const float base = base_of(st.m);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (q + u * TEAM < end) {
#pragma unroll
                for (int e = 0; e < E; ++e) stat_add(st, base, f[u][e]);
            }
    }
    float own[1] = {st.m};                                             // this thread's largest value
    constexpr int WAVE = TEAM < 256 ? TEAM : 64;
    stat_move(st, team_largest<WAVE>(st.m));
    st.s = team_sum<WAVE>(st.s);
    st.t = team_sum<WAVE>(st.t);
    if constexpr (TEAM == 256) {
        if ((tid & 63) == 0) { sh.m[tid >> 6] = st.m; sh.s[tid >> 6] = st.s; sh.t[tid >> 6] = st.t; }
        __syncthreads();
        float m = sh.m[0];
        for (int w = 1; w < 4; ++w) m = fmaxf(m, sh.m[w]);
        Stat sum{m, 0.f, 0.f};
        for (int w = 0; w < 4; ++w) {
            Stat p{sh.m[w], sh.s[w], sh.t[w]};
            stat_move(p, m);
            sum.s += p.s;
            sum.t += p.t;
        }
        st = sum;
    }
    const bool whole = a.segments == 1;
    u64* part = whole ? nullptr : a.parts + (i * a.segments + seg) * (2 + a.k);
    const float base = base_of(st.m), logs = logf(st.s);
    if (tid == 0) {
        if (whole) lp_finish(a, target, i, st, logs);
        else {
            part[0] = ((u64)__float_as_uint(st.s) << 32) | __float_as_uint(st.m);
            part[1] = __float_as_uint(st.t);
        }
    }
    if constexpr (TOP) {
        auto put = [&](int k, u64 r) {                                 // alternative k, by one thread
            if (whole) {
                a.top[i * a.k + k] = (rank_value(r) - base) - logs;
                a.top_index[i * a.k + k] = rank_index(r);
            } else {
                part[2 + k] = r;
            }
        };
        bool slow = st.s != st.s;                                      // the same for the whole team, as all that follows
        if (!slow) {
            if (tid == 0) sh.ncand = 0;
            auto collect = [&](const float* v, int q, float least) {   // the order has no effect: the ranks decide
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int c = q * E - off + e;
                    if (v[e] >= least && c >= 0 && c < a.C) {
                        const int at = atomicAdd(&sh.ncand, 1);
                        if (at < TeamShared<TEAM>::CAND) sh.cand[at] = rank_of(v[e], c);
                    }
                }
            };
            if constexpr (TEAM < 256) {
                const float least = kth_largest<TEAM, 1>(own, a.k, tid);
                team_sync<TEAM>();
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (q0 + tid + u * TEAM < q1) collect(f[u], q0 + tid + u * TEAM, least);
            } else {
                sh.max[tid] = own[0];
                if (tid == 0) sh.winners = 0;
                __syncthreads();
                if (tid < 64) {
                    float v[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) v[w] = sh.max[w * 64 + tid];
                    const float least = kth_largest<64, 4>(v, a.k, tid);
                    if (tid == 0) sh.least = least;
                }
                __syncthreads();
                const float least = sh.least;
                if (own[0] >= least && q0 + tid < q1) sh.winner[atomicAdd(&sh.winners, 1)] = tid;
                __syncthreads();
                const int each = (q1 - q0 + TEAM - 1) / TEAM, n = sh.winners;
                for (int p = tid; p < n * each; p += TEAM) {
                    const int q = q0 + sh.winner[p / each] + p % each * TEAM;
                    if (q >= q1) continue;
                    float v[E];
                    chunk_values<T>(load_chunk(span, row, off, a.C, q), v);
                    collect(v, q, least);
                }
            }
            team_sync<TEAM>();
            const int n = sh.ncand;
            slow = n > TeamShared<TEAM>::CAND;
            if (!slow) {
                for (int c = tid; c < n; c += TEAM) {
                    const u64 r = sh.cand[c];
                    const int before = count_above(sh.cand, n, r);
                    if (before < a.k) put(before, r);
                }
                for (int k = n + tid; k < a.k; k += TEAM) put(k, 0);   // a segment of fewer classes
            }
        }
        if (slow) {
            u64 last = ~0ull;
            for (int k = 0; k < a.k; ++k) {
                last = team_round<T, TEAM>(sh, row, off, a.C, q0, q1, tid, last);
                if (tid == 0) put(k, last);
            }
        }
    }
}

// The segments of a row joined by one workgroup: their alternatives meet in LDS and find their places by counting, or, where they
// are many, by rounds
#define JOIN 1024
template <typename T>
__global__ __launch_bounds__(256) void lp_join_kernel(const LpArgs a) {
    __shared__ float m4[4], s4[4], t4[4];
    __shared__ u64 cand[JOIN];
    const long long i = blockIdx.x;
    const int step = 2 + a.k, tid = threadIdx.x, n = a.segments * a.k;
    const u64* part = a.parts + i * a.segments * step;
    LpTarget target{};
    if (tid == 0) target = lp_target(a, (const T*)a.z + i * a.sn, i);
    for (int c = tid; c < n && c < JOIN; c += 256) cand[c] = part[(long long)(c / a.k) * step + 2 + c % a.k];
    Stat st{-INFINITY, 0.f, 0.f};
    for (int g = tid; g < a.segments; g += 256) {
        const u64 ms = part[(long long)g * step];
        Stat p{__uint_as_float((unsigned)ms), __uint_as_float((unsigned)(ms >> 32)), __uint_as_float((unsigned)part[(long long)g * step + 1])};
        const float m = fmaxf(p.m, st.m);
        stat_move(st, m);
        stat_move(p, m);
        st.s += p.s;
        st.t += p.t;
    }
    stat_move(st, team_largest<64>(st.m));
    st.s = team_sum<64>(st.s);
    st.t = team_sum<64>(st.t);
    if ((tid & 63) == 0) { m4[tid >> 6] = st.m; s4[tid >> 6] = st.s; t4[tid >> 6] = st.t; }
    __syncthreads();
    st = Stat{fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), 0.f, 0.f};
    for (int w = 0; w < 4; ++w) {
        Stat p{m4[w], s4[w], t4[w]};
        stat_move(p, st.m);
        st.s += p.s;
        st.t += p.t;
    }
    const float logs = logf(st.s), base = base_of(st.m);
    if (tid == 0) lp_finish(a, target, i, st, logs);
    auto put = [&](int k, u64 r) {
        a.top[i * a.k + k] = (rank_value(r) - base) - logs;
        a.top_index[i * a.k + k] = rank_index(r);
    };
    if (n <= JOIN) {
        for (int c = tid; c < n; c += 256) {
            const u64 r = cand[c];
            const int before = count_above(cand, n, r);
            if (r && before < a.k) put(before, r);                     // 0: a segment of fewer classes
        }
        return;
    }
    u64 last = ~0ull;
    for (int k = 0; k < a.k && tid < 64; ++k) {
        u64 r = 0;
        for (int c = tid; c < n; c += 64) {
            const u64 o = part[(long long)(c / a.k) * step + 2 + c % a.k];
            r = o < last && o > r ? o : r;
        }
        last = team_best<64>(r);
        if (tid == 0) put(k, last);
    }
}

// Many rows of few classes that lie one behind the other: 256 rows are brought to LDS as one stretch of memory, and a thread works off
// a row there, once for the maximum and once for the sums.  Rows of an even number of classes are begun at another class in each lane,
// which spreads the lanes over LDS's banks.  Alternatives as in lp_position_kernel, equal values by their classes.
#define LDS_ROW 160       // bytes of a row at most: 4 workgroups fit a CU's LDS
template <typename T>
__device__ __forceinline__ void rows_to_lds(const T* z, int count, i32x4* stage) {
    constexpr int E = Elem<T>::EPC;
    for (int q = threadIdx.x; q < count / E; q += 256) stage[q] = ((const i32x4*)z)[q];
    for (int e = count / E * E + threadIdx.x; e < count; e += 256) ((T*)stage)[e] = z[e];
}
template <typename T, int KT>
__global__ __launch_bounds__(256) void lp_rows_lds_kernel(const LpArgs a) {
    constexpr int K = KT > 0 ? KT : 1;
    extern __shared__ i32x4 stage[];
    const long long first = (long long)blockIdx.x * 256, i = first + threadIdx.x;
    rows_to_lds<T>((const T*)a.z + first * a.C, (int)(a.N - first < 256 ? a.N - first : 256) * a.C, stage);
    __syncthreads();
    if (i >= a.N) return;
    const T* row = (const T*)stage + threadIdx.x * a.C;
    const int begin = a.C % 2 ? 0 : threadIdx.x % a.C;
    const LpTarget target = lp_target(a, row, i);
    Stat st{-INFINITY, 0.f, 0.f};
    for (int c = 0; c < a.C; ++c) st.m = fmaxf(st.m, Elem<T>::ld(row + (c + begin < a.C ? c + begin : c + begin - a.C)));
    const float base = base_of(st.m);
    float tv[K];
    int tc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) { tv[k] = -INFINITY; tc[k] = -1; }
    for (int n = 0; n < a.C; ++n) {
        const int c = n + begin < a.C ? n + begin : n + begin - a.C;
        const float z = Elem<T>::ld(row + c);
        stat_add(st, base, z);
        if (KT > 0) {
            bool up[K];
#pragma unroll
            for (int k = 0; k < K; ++k) up[k] = z > tv[k] || (z == tv[k] && c < tc[k]);
#pragma unroll
            for (int k = K - 1; k >= 0; --k) {
                const bool from_above = k > 0 && up[k > 0 ? k - 1 : 0];
                tv[k] = from_above ? tv[k > 0 ? k - 1 : 0] : up[k] ? z : tv[k];
                tc[k] = from_above ? tc[k > 0 ? k - 1 : 0] : up[k] ? c : tc[k];
            }
        }
    }
    const float logs = logf(st.s);
    lp_finish(a, target, i, st, logs);
    if (KT == 0) return;
    bool rounds = logs != logs;
#pragma unroll
    for (int k = 0; k < K; ++k) rounds = rounds || (k < a.k && tc[k] < 0);
    if (!rounds) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < a.k) {
                a.top[i * a.k + k] = (tv[k] - base) - logs;
                a.top_index[i * a.k + k] = tc[k];
            }
        return;
    }
    u64 last = ~0ull;
    for (int k = 0; k < a.k; ++k) {
        u64 best = 0;
        for (int c = 0; c < a.C; ++c) {
            const u64 r = rank_of(Elem<T>::ld(row + c), c);
            best = r < last && r > best ? r : best;
        }
        last = best;
        a.top[i * a.k + k] = (rank_value(best) - base) - logs;
        a.top_index[i * a.k + k] = rank_index(best);
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
    long long first;                   // rows: the launch's first one
};

// dz_j = -p_j (pull + gh log p_j) for every class, pull = gl + sum gk + gh H; the target and the alternatives get their own terms
// added.  A position whose gradients are all 0 gets 0 whatever its logits hold.
__device__ __forceinline__ float lp_grad(float z, float base, float logs, float gh, float pull) {
    const float lp = (z - base) - logs;
    return -__builtin_amdgcn_exp2f(lp * LOG2E) * fmaf(gh, fmaxf(lp, -200.f), pull);          // p = 0: 0 * -inf
}

// gl of a target that is not ignored: one outside [0, C) has log p = NaN, and so has its gradient unless nothing comes in
__device__ __forceinline__ float target_grad(bool inside, float g) { return inside || g == 0.f ? g : __builtin_nanf(""); }

// One thread per P positions, as in the forward pass (6 x 20 x 512 x 1024 fp32 with 2 alternatives 123 us, 5.3 TB/s).  The target's
// term and those of up to KT alternatives are added on the way; where there are more (KT < 0), the classes that are alternatives are
// written once more.
template <typename T, int P, int KT>
__global__ __launch_bounds__(256) void lp_position_bwd_kernel(const LpBwdArgs a) {
    constexpr int K = KT > 0 ? KT : 1;
    const long long rows = a.N * a.L;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * P; i < rows; i += (long long)gridDim.x * 256 * P) {
        long long n, l;
        split_position(i, a.L, n, l);
        const T* row = (const T*)a.z + n * a.sn + l;
        T* out = (T*)a.dz + n * a.dn + l;
        float gl[P], gh[P], pull[P], base[P], logs[P], gk[K][P];
        int t[P], jk[K][P];
        bool any[P], some = false;
#pragma unroll
        for (int p = 0; p < P; ++p) { gl[p] = gh[p] = 0.f; t[p] = -1; }
        if (a.g_log_prob) {
            load_positions<float, P>(a.g_log_prob + i, gl);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const long long v = a.target[i + p];
                t[p] = v >= 0 && v < a.C ? (int)v : -1;
                gl[p] = v == a.ignore ? 0.f : target_grad(t[p] >= 0, gl[p]);
            }
        }
        if (a.g_entropy) load_positions<float, P>(a.g_entropy + i, gh);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            pull[p] = gl[p];
            any[p] = gl[p] != 0.f || gh[p] != 0.f;
        }
        if (KT > 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int p = 0; p < P; ++p) { gk[k][p] = 0.f; jk[k][p] = -1; }
                if (k < a.k) {
                    load_positions<float, P>(a.g_top + (n * a.k + k) * a.L + l, gk[k]);
                    load_indices<P>(a.top_index + (n * a.k + k) * a.L + l, jk[k]);
#pragma unroll
                    for (int p = 0; p < P; ++p) { pull[p] += gk[k][p]; any[p] = any[p] || gk[k][p] != 0.f; }
                }
            }
        }
        if (KT < 0)
            for (int k = 0; k < a.k; ++k)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const float g = a.g_top[(n * a.k + k) * a.L + l + p];
                    pull[p] += g;
                    any[p] = any[p] || g != 0.f;
                }
        load_positions<float, P>(a.stats + i, base);
        load_positions<float, P>(a.stats + rows + i, logs);
        if (a.g_entropy) {
            float h[P];
            load_positions<float, P>(a.entropy + i, h);
#pragma unroll
            for (int p = 0; p < P; ++p) pull[p] = gh[p] != 0.f ? fmaf(gh[p], h[p], pull[p]) : pull[p];
        }
#pragma unroll
        for (int p = 0; p < P; ++p) some = some || any[p];
        for (int c0 = 0; c0 < a.C; c0 += BATCH) {
            Positions<T, P> raw[BATCH];
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (some && c0 + b < a.C) raw[b] = read_positions<T, P>(row + (c0 + b) * a.sc);
#pragma unroll
            for (int b = 0; b < BATCH; ++b)
                if (c0 + b < a.C) {
                    float f[P], d[P];
                    position_values<T, P>(raw[b], f);
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        float own = t[p] == c0 + b ? gl[p] : 0.f;
                        if (KT > 0) {
#pragma unroll
                            for (int k = 0; k < K; ++k) own += jk[k][p] == c0 + b ? gk[k][p] : 0.f;
                        }
                        d[p] = any[p] ? lp_grad(f[p], base[p], logs[p], gh[p], pull[p]) + own : 0.f;
                    }
                    store_positions<T, P>(out + (c0 + b) * a.dc, d);
                }
        }
        if (KT >= 0) continue;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (!any[p]) continue;
            for (int k = 0; k < a.k; ++k) {
                const long long j = a.top_index[(n * a.k + k) * a.L + l + p];
                if (j < 0 || j >= a.C) continue;                       // no class: pull has its gradient, as in the other kernels
                float own = j == t[p] ? gl[p] : 0.f;
                for (int o = 0; o < a.k; ++o) {
                    const long long at = (n * a.k + o) * a.L + l + p;
                    if (a.top_index[at] == j) own += a.g_top[at];
                }
                Elem<T>::st(out + p + j * a.dc, lp_grad(Elem<T>::ld(row + p + j * a.sc), base[p], logs[p], gh[p], pull[p]) + own);
            }
        }
    }
}

// Many rows of few classes, brought to LDS and back as lp_rows_lds_kernel brings them there
template <typename T, int KT>
__global__ __launch_bounds__(256) void lp_rows_lds_bwd_kernel(const LpBwdArgs a) {
    constexpr int K = KT > 0 ? KT : 1, E = Elem<T>::EPC;
    extern __shared__ i32x4 stage[];
    T* lds = (T*)stage;
    const long long first = (long long)blockIdx.x * 256, i = first + threadIdx.x;
    const int rows = (int)(a.N - first < 256 ? a.N - first : 256), count = rows * a.C;
    const T* z = (const T*)a.z + first * a.C;
    T* dz = (T*)a.dz + first * a.C;
    rows_to_lds<T>(z, count, stage);
    float gl = 0.f, gh = 0.f, pull, base = 0.f, logs = 0.f, gk[K];
    int t = -1, jk[K];
    bool any = false;
    if (i < a.N) {
        if (a.g_log_prob) {
            const long long v = a.target[i];
            t = v >= 0 && v < a.C ? (int)v : -1;
            gl = v == a.ignore ? 0.f : target_grad(t >= 0, a.g_log_prob[i]);
        }
        if (a.g_entropy) gh = a.g_entropy[i];
        base = a.stats[i];
        logs = a.stats[a.N + i];
    }
    pull = gl;
    any = gl != 0.f || gh != 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        gk[k] = 0.f;
        jk[k] = -1;
        if (KT > 0 && k < a.k && i < a.N) {
            gk[k] = a.g_top[i * a.k + k];
            load_indices<1>(a.top_index + i * a.k + k, &jk[k]);
            pull += gk[k];
            any = any || gk[k] != 0.f;
        }
    }
    if (gh != 0.f) pull = fmaf(gh, a.entropy[i], pull);
    __syncthreads();
    if (i < a.N) {
        T* row = lds + threadIdx.x * a.C;
        int c = a.C % 2 ? 0 : threadIdx.x % a.C;
        for (int n = 0; n < a.C; ++n) {
            float own = t == c ? gl : 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) own += KT > 0 && jk[k] == c ? gk[k] : 0.f;
            Elem<T>::st(row + c, any ? lp_grad(Elem<T>::ld(row + c), base, logs, gh, pull) + own : 0.f);
            c = c + 1 == a.C ? 0 : c + 1;
        }
    }
    __syncthreads();
    for (int q = threadIdx.x; q < count / E; q += 256) ((i32x4*)dz)[q] = stage[q];
    for (int e = count / E * E + threadIdx.x; e < count; e += 256) dz[e] = lds[e];
}

// Rows by teams (4096 x 32001 bf16 86 us, 6.1 TB/s: the memory bounds it): chunks at the 16-byte boundaries as in the forward pass;
// the target and the alternatives are written once more after the rest.  A gradient row that lies differently to the boundaries than the logits' row is stored class by class.
#define BWD_UNROLL 4
template <typename T, int TEAM>
__global__ __launch_bounds__(256) void lp_rows_bwd_kernel(const LpBwdArgs a) {
    constexpr int E = Elem<T>::EPC;
    const int tid = threadIdx.x % TEAM;
    const long long i = a.first + (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    if (TEAM < 256 && i >= a.N) return;                                // no barrier of the workgroup below for teams within a wave
    const T* row = (const T*)a.z + i * a.sn;
    T* out = (T*)a.dz + i * a.dn;
    const int off = (int)(((unsigned long long)row / sizeof(T)) % E), dist = (int)(((unsigned long long)out / sizeof(T)) % E);
    const int chunks = (a.C + off + E - 1) / E, q0 = blockIdx.y * TEAM * BWD_UNROLL, q1 = min(q0 + TEAM * BWD_UNROLL, chunks);
    const long long t = a.g_log_prob ? a.target[i] : a.ignore;
    const float gl = t == a.ignore ? 0.f : target_grad(t >= 0 && t < a.C, a.g_log_prob[i]), gh = a.g_entropy ? a.g_entropy[i] : 0.f;
    float pull = gl;
    bool any = gl != 0.f || gh != 0.f;
    // alternative wl + r W is lane wl's of every wave (W lanes of it): its gradient, its class and that class's logit, all on their way
    // before the row (5 of them on 100000 x 1000 bf16: 102 us against 147 where they are looked up afterwards); the target is lane 0's.  Classes of other workgroups, and those outside the row, are -1.
    constexpr int W = TEAM < 64 ? TEAM : 64, R = W < ERF_TOP_MAX ? ERF_TOP_MAX / W : 1;
    const int wl = threadIdx.x % W;
    auto here = [&](long long j) { return j >= 0 && j < a.C && j + off >= (long long)q0 * E && j + off < (long long)q1 * E ? (int)j : -1; };
    const int mine_t = here(t);
    const float zt = tid == 0 && mine_t >= 0 ? Elem<T>::ld(row + mine_t) : 0.f;
    float gk[R], zk[R];
    int jk[R];
    if (a.k) {
        float sum = 0.f, set = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int k = wl + r * W;
            gk[r] = k < a.k ? a.g_top[i * a.k + k] : 0.f;
            jk[r] = k < a.k ? here(a.top_index[i * a.k + k]) : -1;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            zk[r] = tid < W && jk[r] >= 0 ? Elem<T>::ld(row + jk[r]) : 0.f;
            sum += gk[r];
            set += gk[r] != 0.f;
        }
        pull += team_sum<W>(sum);
        any = any || team_sum<W>(set) != 0.f;
    }
    const float base = a.stats[i], logs = a.stats[a.N + i];
    if (gh != 0.f) pull = fmaf(gh, a.entropy[i], pull);
    {
        const int q = q0 + tid;
        const Span<T> span = span_of<T>(a);
        i32x4 raw[BWD_UNROLL];
#pragma unroll
        for (int u = 0; u < BWD_UNROLL; ++u)
            if (any && q + u * TEAM < q1) raw[u] = load_chunk(span, row, off, a.C, q + u * TEAM);
#pragma unroll
        for (int u = 0; u < BWD_UNROLL; ++u) {
            if (q + u * TEAM >= q1) break;
            const int c0 = (q + u * TEAM) * E - off;
            float f[E], d[E];
            chunk_values<T>(raw[u], f);
#pragma unroll
            for (int e = 0; e < E; ++e) d[e] = any ? lp_grad(f[e], base, logs, gh, pull) : 0.f;
            if (c0 >= 0 && c0 + E <= a.C && off == dist) {
                if constexpr (E == 4) *(f32x4*)(out + c0) = f32x4{d[0], d[1], d[2], d[3]};
                else *(i32x4*)(out + c0) = i32x4{pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]), pack_bf16x2(d[6], d[7])};
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (c0 + e >= 0 && c0 + e < a.C) Elem<T>::st(out + c0 + e, d[e]);
            }
        }
    }
    if (!any) return;                                             // the same for the whole team
    // the stores above are done before a class is written again
    if (TEAM < 256) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    else __syncthreads();
    if (tid >= W) return;
    float own_t = gl;
    if (a.k) {
        float own[R];
#pragma unroll
        for (int r = 0; r < R; ++r) own[r] = jk[r] == mine_t ? gl : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)                                    // the same class given twice gets both
            for (int o = 0; o < W && o + r * W < a.k; ++o) {
                const int j = __shfl(jk[r], o, W);
                const float g = __shfl(gk[r], o, W);
                own_t += j == mine_t ? g : 0.f;
#pragma unroll
                for (int v = 0; v < R; ++v) own[v] += j == jk[v] ? g : 0.f;
            }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (jk[r] >= 0) Elem<T>::st(out + jk[r], lp_grad(zk[r], base, logs, gh, pull) + own[r]);
    }
    if (tid == 0 && mine_t >= 0) Elem<T>::st(out + mine_t, lp_grad(zt, base, logs, gh, pull) + own_t);
}

static inline bool lp_shape_ok(int dtype, long long N, int C, long long L, long long sn, long long sc, int k) {
    if ((dtype != ERF_F32 && dtype != ERF_BF16) || N <= 0 || C <= 0 || C > (1 << 28) || L <= 0 || sn < 0 || k < 0 || k > C || k > ERF_TOP_MAX) return false;
    if (N > 0x7FFFFFFFll || L > 0x7FFFFFFFll || N * L > (1ll << 40)) return false;
    return (sc == 1 && L == 1) || (sc >= L && sc >= 2);
}

// Whether no two elements of dlogits share a place: images one behind the other, or images side by side within a class
static inline bool lp_apart(long long N, int C, long long L, long long dn, long long dc) {
    return N == 1 || (__int128)dn >= (__int128)(C - 1) * dc + L || (dn >= L && (__int128)dc >= (__int128)(N - 1) * dn + L);
}

static inline unsigned lp_grid(long long total) {
    const long long g = (total + 255) / 256;
    return (unsigned)(g > 65536 ? 65536 : g);
}

// Positions per thread: 4 where whole vectors lie on their boundaries, enough threads are left to fill the chip and no alternatives
// take up registers.  1 / 4 positions, us, forward and backward: 6 x 20 x 512 x 1024 bf16 46 / 41 and 69 / 69, fp32 64 / 65 and 103 / 111,
// 6 x 5 x 512 x 1024 bf16 22 / 21 and 29 / 25, fp32 26 / 24 and 38 / 37; with 2 alternatives 6 x 20 x 512 x 1024 bf16 66 / 63 and 87 / 96,
// fp32 80 / 83 and 119 / 126.
static inline int lp_positions(int dtype, long long N, long long L, long long sc, unsigned long long addresses, unsigned long long strides,
                               unsigned long long per_position, int k) {
    const int size = dtype == ERF_BF16 ? 2 : 4;
    return sc != 1 && L % 4 == 0 && strides % 4 == 0 && addresses % (4 * size) == 0 && per_position % 16 == 0 && N * L >= (1ll << 19) && !k ? 4 : 1;
}

// Rows of more classes than a thread walks through by itself are taken by the smallest team that has the whole row in registers
// wherever it starts (and lanes for the alternatives), or by a workgroup.  8 chunks a thread let a smaller team have a row, fewer
// waves stay on a SIMD: forward, 8 / 4 chunks, 100000 x 1000 bf16 42 / 65 us, 20000 x 2049 25 / 39, 100000 x 200 15 / 13, 20000 x 2000
// 23 / 19: 8 where 4 would need the larger team.  Few rows of very many classes are split so that about 1024 workgroups have work.
static inline int lp_epc(int dtype) { return dtype == ERF_BF16 ? 8 : 4; }
// A thread takes a whole row of up to `alone` classes: up to there a wave's rows fill the cache lines that its loads touch.  1000000
// rows by threads / by teams, us: forward fp32 24 classes 59 / 53, 32 88 / 54, bf16 40 51 / 75, 48 101 / 80; with 2 alternatives fp32 32
// 90 / 90, 40 129 / 107, bf16 56 99 / 129, 64 162 / 127; backward fp32 12 49 / 51, 16 88 / 57; bf16 12 27 / 68, 16 55 / 48, 24 91 / 48.
#define ALONE_FWD(dtype, k) ((dtype) == ERF_BF16 ? ((k) ? 56 : 44) : ((k) ? 32 : 24))
#define ALONE_BWD 12
struct LpTeam { int team, each; };     // team 1: a thread; each: chunks in flight per thread
static inline LpTeam lp_team(int dtype, int C, int k, int alone, int most) {
    static const LpTeam teams[] = {{8, 4}, {16, 4}, {16, 8}, {64, 4}, {64, 8}};
    if (C <= alone) return {1, 0};
    for (const LpTeam& t : teams)
        if (t.each <= most && k <= t.team && C <= (t.team * t.each - 1) * lp_epc(dtype) + 1) return t;
    return {256, 4};
}
static inline LpTeam lp_fwd_team(int dtype, int C, int k) { return lp_team(dtype, C, k, ALONE_FWD(dtype, k), 8); }
static inline LpTeam lp_bwd_team(int dtype, int C) { return lp_team(dtype, C, 0, ALONE_BWD, BWD_UNROLL); }
static inline int lp_segments(int dtype, long long N, int C, int k) {
    if (lp_fwd_team(dtype, C, k).team < 256) return 1;
    const long long most = ((long long)C + 1024 * lp_epc(dtype) - 1) / (1024 * lp_epc(dtype)), want = (1024 + N - 1) / N;
    return (int)(want < most ? want : most);
}

// Rows through LDS: compact, on 16-byte boundaries, few enough classes that 4 workgroups fit a CU's LDS, enough rows to fill the chip.
// LDS against threads or teams, us, backward: 3145728 x 20 fp32 115 / 248, bf16 68 / 275; 1000000 x 9 18 / 30 and 13 / 18; 1000000 x 24 41
// / 75 and 24 / 48; with 5 alternatives 61 / 118 and 42 / 72; 65536 x 20 5.7 / 6.8 and 5.2 / 6.4.  Forward, from 13 classes on: 3145728 x 20
// 69 / 124 and 49 / 65, 1000000 x 9 14 / 13 and 12 / 13, 1000000 x 32 37 / 53 and 26 / 60; with 2 alternatives 55 / 91 and 36 / 63,
// with 5 113 / 106 and 83 / 77.
static inline bool lp_in_lds(int dtype, long long N, int C, long long sn, long long sc, int k, int most_k, unsigned long long addresses) {
    return sc == 1 && sn == C && addresses % 16 == 0 && C * (dtype == ERF_BF16 ? 2 : 4) <= LDS_ROW && N >= (1 << 16) && k <= most_k;
}

// A launch has less than 2^32 threads: very many rows are several launches' work
#define ROWS_PER_LAUNCH(team) ((1ll << 30) / (team))

template <typename T, bool TOP>
static void lp_rows_launch(LpArgs a, int dtype, hipStream_t s) {
    const auto [team, each] = lp_fwd_team(dtype, a.C, a.k);
    for (a.first = 0; a.first < a.N; a.first += ROWS_PER_LAUNCH(team)) {
        const long long rows = a.N - a.first < ROWS_PER_LAUNCH(team) ? a.N - a.first : ROWS_PER_LAUNCH(team);
        const dim3 grid((unsigned)((rows * team + 255) / 256), (unsigned)a.segments), block(256);
        if (team == 8) hipLaunchKernelGGL((lp_rows_kernel<T, 8, 4, TOP>), grid, block, 0, s, a);
        else if (team == 16 && each == 4) hipLaunchKernelGGL((lp_rows_kernel<T, 16, 4, TOP>), grid, block, 0, s, a);
        else if (team == 16) hipLaunchKernelGGL((lp_rows_kernel<T, 16, 8, TOP>), grid, block, 0, s, a);
        else if (team == 64 && each == 4) hipLaunchKernelGGL((lp_rows_kernel<T, 64, 4, TOP>), grid, block, 0, s, a);
        else if (team == 64) hipLaunchKernelGGL((lp_rows_kernel<T, 64, 8, TOP>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((lp_rows_kernel<T, 256, 4, TOP>), grid, block, 0, s, a);
    }
    if (a.segments > 1) hipLaunchKernelGGL(lp_join_kernel<T>, dim3((unsigned)a.N), dim3(256), 0, s, a);
}

template <typename T>
static void lp_rows_bwd_launch(LpBwdArgs a, int dtype, hipStream_t s) {
    const int team = lp_bwd_team(dtype, a.C).team, per = 256 * BWD_UNROLL;
    const int chunks = (a.C + 2 * (lp_epc(dtype) - 1)) / lp_epc(dtype);              // of a row that starts just before a boundary
    for (a.first = 0; a.first < a.N; a.first += ROWS_PER_LAUNCH(team)) {
        const long long rows = a.N - a.first < ROWS_PER_LAUNCH(team) ? a.N - a.first : ROWS_PER_LAUNCH(team);
        const dim3 grid((unsigned)((rows * team + 255) / 256), team < 256 ? 1u : (unsigned)((chunks + per - 1) / per)), block(256);
        if (team == 8) hipLaunchKernelGGL((lp_rows_bwd_kernel<T, 8>), grid, block, 0, s, a);
        else if (team == 16) hipLaunchKernelGGL((lp_rows_bwd_kernel<T, 16>), grid, block, 0, s, a);
        else if (team == 64) hipLaunchKernelGGL((lp_rows_bwd_kernel<T, 64>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((lp_rows_bwd_kernel<T, 256>), grid, block, 0, s, a);
    }
}

extern "C" {

size_t erf_class_log_probs_workspace_bytes(int dtype, long long N, int C, long long L, long long stride_c, int top_k) {
    if (!lp_shape_ok(dtype, N, C, L, 0, stride_c, top_k) || stride_c != 1) return 0;
    const int segments = lp_segments(dtype, N, C, top_k);
    return segments > 1 ? (size_t)N * segments * (2 + top_k) * sizeof(u64) : 0;
}

int erf_class_log_probs_fwd(const void* logits, int dtype, long long N, int C, long long L, long long stride_n, long long stride_c,
                            const long long* target, long long ignore_index, float* log_prob, float* entropy, float* stats, int top_k,
                            float* top_log_probs, long long* top_indices, void* workspace, void* stream) {
    if (!logits || !entropy || (!target != !log_prob) || !lp_shape_ok(dtype, N, C, L, stride_n, stride_c, top_k) ||
        (top_k && (!top_log_probs || !top_indices)) ||
        (!workspace && erf_class_log_probs_workspace_bytes(dtype, N, C, L, stride_c, top_k)))
        return ERF_EINVAL;
    LpArgs a{logits, target, N, L, stride_n, stride_c, C, top_k, ignore_index, log_prob, entropy, stats, top_log_probs, top_indices, 1, 0, (u64*)workspace};
    hipStream_t s = (hipStream_t)stream;
    if (C > 12 && lp_in_lds(dtype, N, C, stride_n, stride_c, top_k, 2, (unsigned long long)logits)) {
        const dim3 grid((unsigned)((N + 255) / 256)), block(256);
        const size_t lds = (size_t)256 * C * (dtype == ERF_BF16 ? 2 : 4);
#define LP_KT(T)                                                                                            \
    do {                                                                                                    \
        if (top_k == 0) hipLaunchKernelGGL((lp_rows_lds_kernel<T, 0>), grid, block, lds, s, a);             \
        else hipLaunchKernelGGL((lp_rows_lds_kernel<T, 2>), grid, block, lds, s, a);                        \
    } while (0)
        if (dtype == ERF_BF16) LP_KT(bf16raw); else LP_KT(float);
#undef LP_KT
    } else if (stride_c == 1 && lp_fwd_team(dtype, C, top_k).team > 1) {
        a.segments = lp_segments(dtype, N, C, top_k);
        if (dtype == ERF_BF16) { if (top_k) lp_rows_launch<bf16raw, true>(a, dtype, s); else lp_rows_launch<bf16raw, false>(a, dtype, s); }
        else { if (top_k) lp_rows_launch<float, true>(a, dtype, s); else lp_rows_launch<float, false>(a, dtype, s); }
    } else {
        const int p = lp_positions(dtype, N, L, stride_c, (unsigned long long)logits, (unsigned long long)(stride_n | stride_c),
                                   (unsigned long long)log_prob | (unsigned long long)entropy | (unsigned long long)stats, top_k);
        const dim3 grid(lp_grid(N * L / p)), block(256);
#define LP_KT(T)                                                                                            \
    do {                                                                                                    \
        if (p == 4) hipLaunchKernelGGL((lp_position_kernel<T, 4, 0>), grid, block, 0, s, a);                \
        else if (top_k == 0) hipLaunchKernelGGL((lp_position_kernel<T, 1, 0>), grid, block, 0, s, a);       \
        else if (top_k == 1) hipLaunchKernelGGL((lp_position_kernel<T, 1, 1>), grid, block, 0, s, a);       \
        else if (top_k == 2) hipLaunchKernelGGL((lp_position_kernel<T, 1, 2>), grid, block, 0, s, a);       \
        else if (top_k <= 4) hipLaunchKernelGGL((lp_position_kernel<T, 1, 4>), grid, block, 0, s, a);       \
        else if (top_k <= 8) hipLaunchKernelGGL((lp_position_kernel<T, 1, 8>), grid, block, 0, s, a);       \
        else hipLaunchKernelGGL((lp_position_kernel<T, 1, -1>), grid, block, 0, s, a);                      \
    } while (0)
        if (dtype == ERF_BF16) LP_KT(bf16raw); else LP_KT(float);
#undef LP_KT
    }
    return erf_check_launch();
}

int erf_class_log_probs_bwd(const void* logits, int dtype, long long N, int C, long long L, long long stride_n, long long stride_c,
                            const long long* target, long long ignore_index, const float* stats, const float* entropy,
                            const float* g_log_prob, const float* g_entropy, int top_k, const long long* top_indices, const float* g_top,
                            void* dlogits, long long dstride_n, long long dstride_c, void* stream) {
    if (!logits || !stats || !entropy || !dlogits || (g_log_prob && !target) || !lp_shape_ok(dtype, N, C, L, stride_n, stride_c, top_k) ||
        (g_top && (!top_indices || !top_k)) || dstride_n < 0 || (dstride_c == 1) != (stride_c == 1) || (dstride_c != 1 && dstride_c < L) ||
        !lp_apart(N, C, L, dstride_n, dstride_c))
        return ERF_EINVAL;
    const LpBwdArgs a{logits, target, N, L, stride_n, stride_c, dstride_n, dstride_c, C, g_top ? top_k : 0, ignore_index, stats, entropy,
                      g_log_prob, g_entropy, g_top, top_indices, dlogits, 0};
    hipStream_t s = (hipStream_t)stream;
    if (lp_in_lds(dtype, N, C, stride_n, stride_c, a.k, 8, (unsigned long long)logits | (unsigned long long)dlogits) && dstride_n == C) {
        const dim3 grid((unsigned)((N + 255) / 256)), block(256);
        const size_t lds = (size_t)256 * C * (dtype == ERF_BF16 ? 2 : 4);
#define LP_KT(T)                                                                                            \
    do {                                                                                                    \
        if (a.k == 0) hipLaunchKernelGGL((lp_rows_lds_bwd_kernel<T, 0>), grid, block, lds, s, a);           \
        else if (a.k <= 2) hipLaunchKernelGGL((lp_rows_lds_bwd_kernel<T, 2>), grid, block, lds, s, a);      \
        else hipLaunchKernelGGL((lp_rows_lds_bwd_kernel<T, 8>), grid, block, lds, s, a);                    \
    } while (0)
        if (dtype == ERF_BF16) LP_KT(bf16raw); else LP_KT(float);
#undef LP_KT
    } else if (stride_c == 1 && lp_bwd_team(dtype, C).team > 1) {
        if (dtype == ERF_BF16) lp_rows_bwd_launch<bf16raw>(a, dtype, s);
        else lp_rows_bwd_launch<float>(a, dtype, s);
    } else {
        const int p = lp_positions(dtype, N, L, stride_c, (unsigned long long)logits | (unsigned long long)dlogits,
                                   (unsigned long long)(stride_n | stride_c | dstride_n | dstride_c),
                                   (unsigned long long)stats | (unsigned long long)entropy | (unsigned long long)g_log_prob |
                                       (unsigned long long)g_entropy, a.k);
        const dim3 grid(lp_grid(N * L / p)), block(256);
#define LP_KT(T)                                                                                            \
    do {                                                                                                    \
        if (p == 4) hipLaunchKernelGGL((lp_position_bwd_kernel<T, 4, 0>), grid, block, 0, s, a);            \
        else if (a.k == 0) hipLaunchKernelGGL((lp_position_bwd_kernel<T, 1, 0>), grid, block, 0, s, a);     \
        else if (a.k <= 2) hipLaunchKernelGGL((lp_position_bwd_kernel<T, 1, 2>), grid, block, 0, s, a);     \
        else if (a.k <= 4) hipLaunchKernelGGL((lp_position_bwd_kernel<T, 1, 4>), grid, block, 0, s, a);     \
        else if (a.k <= 8) hipLaunchKernelGGL((lp_position_bwd_kernel<T, 1, 8>), grid, block, 0, s, a);     \
        else hipLaunchKernelGGL((lp_position_bwd_kernel<T, 1, -1>), grid, block, 0, s, a);                  \
    } while (0)
        if (dtype == ERF_BF16) LP_KT(bf16raw); else LP_KT(float);
#undef LP_KT
    }
    return erf_check_launch();
}

}  // extern "C"
