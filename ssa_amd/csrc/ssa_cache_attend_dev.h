// ssa_cache_attend_dev.h -- what the attention kernels over the paged cache share.
#pragma once

#include "ssa_cache_dev.h"

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

constexpr int ATT_WAVES = 4;                  // of a workgroup
constexpr float LOG2E = 1.44269504088896340736f;

// How a launch's units (groups of CT columns: query rows of one request and kv
// head) are numbered.
enum {
    UNITS_PAGES,    // unit = row and group of its heads
    UNITS_ALL,      // every request's groups
    UNITS_FEW,      // those of requests with at most `many` columns, numbered by request
    UNITS_MANY,     // those of the others
};

struct AttendParams {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *starts, *requests, *positions, *pages;
    const void *q;
    void *out;
    float *part_ml, *part_o;                  // (T * Hq, s_stride, 2), (T * Hq, s_stride, D)
    int64_t num_pages, table_stride, q_st, q_sh, o_st, o_sh;
    int32_t T, R, width, Hq, Hkv, rep, d, page_shift, top, S, s_stride, chunk, mode, many, units;
    int32_t q_vec, o_vec;                     // rows of q in 16-byte pieces, of out in 4 elements
    float scale;                              // softmax scale * log2(e)
};

struct Unit {
    int req, t0, c0, c1;    // row t0 + c / rep, head c % rep, for c in [c0, c1)
};

// The columns of unit u, false if there are none.  Requests' units are numbered
// without a list: in UNITS_ALL and UNITS_MANY request r (R stands for the rows
// behind the last one) has its units from floor(starts[r] rep / CT) + r on, which
// leaves each request ceil(rows rep / CT); found by binary search.
__device__ __forceinline__ bool locate_unit(const AttendParams &p, int u, int CT, Unit &x) {
    if (p.mode == UNITS_PAGES) {
        const int tiles = (p.rep + CT - 1) / CT;
        x.t0 = u / tiles;
        x.c0 = (u - x.t0 * tiles) * CT;
        x.c1 = min(x.c0 + CT, p.rep);
        x.req = p.requests[x.t0];
    } else {
        int lo = 0;
        int64_t j;
        if (p.mode == UNITS_FEW) {
            const int tiles = (p.many + CT - 1) / CT;
            lo = u / tiles;
            j = u - lo * tiles;
            x.t0 = p.starts[lo];
        } else {
            // last r whose first unit is <= u: the wave tests 64 places of lo .. hi at
            // once, so that 64 requests take one load and 4,096 two
            int hi = p.R;
            const int lane = lane_id();
            while (lo < hi) {
                const int step = (hi - lo + SSA_WAVE - 1) / SSA_WAVE;
                const int at = lo + (lane + 1) * step;
                const bool t = at <= hi && (int64_t)p.starts[at] * p.rep / CT + at <= u;
                const uint64_t m = wave_ballot(t);
                const int k = m == ~0ull ? SSA_WAVE : __ffsll((unsigned long long)~m) - 1;
                lo += k * step;
                hi = min(hi, lo + step - 1);
            }
            x.t0 = p.starts[lo];
            j = u - ((int64_t)x.t0 * p.rep / CT + lo);
        }
        const int end = lo < p.R ? p.starts[lo + 1] : p.T;
        const int64_t cols = (int64_t)(min(end, p.T) - x.t0) * p.rep;
        if (x.t0 < 0 || j < 0 || j * CT >= cols) return false;
        if (p.mode == UNITS_FEW && cols > p.many) return false;
        if (p.mode == UNITS_MANY && cols <= p.many) return false;
        x.c0 = (int)(j * CT);
        x.c1 = (int)min((int64_t)x.c0 + CT, cols);
        x.req = lo < p.R ? lo : -1;
    }
    if (x.req >= p.R) x.req = -1;
    return true;
}

// eight codes (two words) times a power of two, as 16-bit floats: exact (a code has
// 4 significant bits; f16 holds all of them unscaled)
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w0, uint32_t w1, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f16x8 codes_f16(uint32_t w0, uint32_t w1) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A matrix operand's lane l holds row l % 16 and piece l / 16 of its columns, so
// neighbouring lanes' pieces lie a whole row apart, and the L1 serves 16 bytes of a
// row an access where it could serve 64 (measured: 45 accesses a load, its data path
// 93% busy at 11 TB/s).  Loads therefore go out with piece l % 4 of row l / 4, and the
// pieces change lanes through LDS: they are written to slot_of(row, piece), read back
// from slot_of(own row, own piece).  The exclusive or keeps 16-byte accesses free of
// bank conflicts (counted): writes go 8 neighbouring lanes at a time, two rows' four
// pieces; reads 16 at a time, half of them 4 lanes in every 12 of one piece, the rest
// their complement in the next.
__device__ __forceinline__ int slot_of(int row, int piece) { return piece * 16 + (row ^ (piece << 1)); }

// Matrix operands by the queries' type.  Queries are exact: bf16, f16, or three bf16
// terms of an fp32.  Probabilities: f16, or three bf16 terms.
template <typename T> struct Ops {                      // bf16
    typedef bf16x8 Q;
    typedef f16x8 P;
    typedef __bf16 QE;
    typedef _Float16 PE;
    static constexpr int NQ = 1, NP = 1;
    static __device__ __forceinline__ Q key(uint32_t a, uint32_t b) { return codes_bf16(a, b, 1.f); }
    static __device__ __forceinline__ P value(uint32_t a, uint32_t b, float) { return codes_f16(a, b); }
};
template <> struct Ops<f16_t> {
    typedef f16x8 Q;
    typedef f16x8 P;
    typedef _Float16 QE;
    typedef _Float16 PE;
    static constexpr int NQ = 1, NP = 1;
    static __device__ __forceinline__ Q key(uint32_t a, uint32_t b) { return codes_f16(a, b); }
    static __device__ __forceinline__ P value(uint32_t a, uint32_t b, float) { return codes_f16(a, b); }
};
template <> struct Ops<float> {
    typedef bf16x8 Q;
    typedef bf16x8 P;
    typedef __bf16 QE;
    typedef __bf16 PE;
    static constexpr int NQ = 3, NP = 3;
    static __device__ __forceinline__ Q key(uint32_t a, uint32_t b) { return codes_bf16(a, b, 1.f); }
    static __device__ __forceinline__ P value(uint32_t a, uint32_t b, float s) { return codes_bf16(a, b, s); }
};

// One wave's columns: queries, running softmax and sums, for tiles of KT keys whose
// scores it is given as S^T (block b, row 4g + r: key KT/4 g + 4b + r).
//
// Per score the vector unit does a maximum, a fused multiply-add, an exponential and
// half a conversion; everything else is kept off that path:
//  * the key scale of a page goes into the multiply-add's constant, the value scale
//    2^e_v into its addend: O is kept in units of 2^e_ref and p_j 2^(e_v - e_ref) is
//    what multiplies the unscaled codes;
//  * sums of p come from the matrix unit, as one more row of V^T (the power of two
//    that undoes these units, so that they are the sums of p as rounded);
//  * O is rescaled only when a column's maximum has grown by more than 2^4, or
//    e_v - e_ref has left 0 .. 6; with 2^5 to spare below, p 2^5 2^(e_v - e_ref) as an
//    f16 stays under 2^15 and its rounding at 11 bits, or 2^-30 of the largest p.
// For fp32 queries p is three bf16 terms (24 bits; V scaled, as bf16 holds every
// scale).
template <typename T, int D, int KT, int RT>
struct Columns {
    typedef Ops<T> O_;
    typedef typename O_::Q QV;
    typedef typename O_::P PV;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int NQ = O_::NQ, NP = O_::NP;
    static constexpr int NB = KT / 16, DP = D / 64, ND = D / 16, KS = KT / 32;
    // p is kept 2^ROOM larger, O in units of 2^(e_ref - ROOM)
    static constexpr float ROOM = F32 ? 0.f : 5.f, GROWN = 4.f, LIFT = 6.f;

    QV q[RT][DP * 2][NQ];
    f32x4 o[RT][ND], l[RT];
    float m[RT], e_ref, scale;
    int pos[RT];                 // last key a column sees; none for it to lose if it is dead
    int most, least;             // of the live columns

    // columns c0 + 16 rt + lane % 16 below c1 of unit u, kv head h
    __device__ __forceinline__ void start(const AttendParams &p, const Unit &u, int c0, int c1, int h) {
        const int lane = lane_id(), col = lane & 15, g = lane >> 4;
        const bool neg = p.scale < 0.f;
        scale = fabsf(p.scale);
        e_ref = 0.f;
        most = -1;
        least = 0x7fffffff;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int c = c0 + rt * 16 + col;
            const bool live = c < c1;
            // dead lanes load the last live column, so that no load waits for another
            const int cc = min(c, c1 - 1), t = u.t0 + cc / p.rep;
            const int32_t req = p.requests[t], at = p.positions[t];
            const int seen = live && u.req >= 0 && req == u.req ? at : -1;
            most = max(most, seen);
            if (live) least = min(least, seen);
            pos[rt] = live ? seen : 0x7fffffff;
            const T *row = (const T *)p.q + t * p.q_st + (int64_t)(h * p.rep + cc % p.rep) * p.q_sh;
            T raw[DP * 2][8];
            if (p.q_vec) {
#pragma unroll
                for (int s = 0; s < DP * 2; ++s) {
                    const int x = (s >> 1) * 64 + g * 16 + (s & 1) * 8;
                    __builtin_memcpy(raw[s], __builtin_assume_aligned(row + (x < p.d ? x : 0), 16),
                                     sizeof(raw[s]));
                }
            } else {
#pragma unroll
                for (int s = 0; s < DP * 2; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        raw[s][j] = row[min((s >> 1) * 64 + g * 16 + (s & 1) * 8 + j, p.d - 1)];
            }
#pragma unroll
            for (int s = 0; s < DP * 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int x = (s >> 1) * 64 + g * 16 + (s & 1) * 8 + j;
                    float v = to_f32(raw[s][j]);
                    v = live && x < p.d ? (neg ? -v : v) : 0.f;
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        const typename O_::QE b = (typename O_::QE)v;
                        q[rt][s][n][j] = b;
                        v -= (float)b;
                    }
                }
            m[rt] = -INFINITY;
            l[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < ND; ++i) o[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        most = (int)wave_max_u((uint32_t)(most + 1)) - 1;
        most = min(most, (p.width << p.page_shift) - 1);
        least = (int)wave_min_u((uint32_t)(least + 1)) - 1;
    }

    // scores to probabilities: key scale ks, value scale vs, first key of the tile;
    // l takes their sums
    __device__ __forceinline__ void softmax(f32x4 (&s)[RT][NB], float ks, float vs, int key0,
                                            PV (&pf)[RT][KS][NP]) {
        const int g = lane_id() >> 4;
        float c = scale * ks;                 // log2 units of a score's unit
        if (key0 + KT - 1 > least) {          // some column ends in this tile
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        s[rt][b][r] = key0 + KT / 4 * g + 4 * b + r <= pos[rt] ? s[rt][b][r] * c
                                                                              : -INFINITY;
            c = 1.f;
        }
        const float ev = F32 ? 0.f : (float)((int)(__float_as_uint(vs) >> 23) - 127);
        float mx[RT];
        bool grow = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float v = s[rt][0][0];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) v = fmaxf(v, s[rt][b][r]);
            mx[rt] = v * c;
            grow |= mx[rt] > m[rt] + GROWN;
        }
        if (wave_ballot(grow) || ev < e_ref || ev > e_ref + LIFT) {
            const float e_new = F32 ? 0.f : ev - 3.f;
            const float unit = __builtin_amdgcn_exp2f(e_ref - e_new);
            e_ref = e_new;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float v = mx[rt];
                v = fmaxf(v, __shfl_xor(v, 16, SSA_WAVE));
                v = fmaxf(v, __shfl_xor(v, 32, SSA_WAVE));
                v = fmaxf(v, m[rt]);
                const float a = __builtin_amdgcn_exp2f(m[rt] - (v == -INFINITY ? 0.f : v));
                m[rt] = v;
                l[rt] *= a;
                const float au = a * unit;
#pragma unroll
                for (int i = 0; i < ND; ++i) o[rt][i] *= au;
            }
        }
        const float lift = ev - e_ref + ROOM;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float sub = lift - (m[rt] == -INFINITY ? 0.f : m[rt]);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = __builtin_amdgcn_exp2f(fmaf(s[rt][b][r], c, sub));
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const typename O_::PE e = (typename O_::PE)v;
                        pf[rt][b >> 1][n][(b & 1) * 4 + r] = e;
                        if (n + 1 < NP) v -= (float)e;
                    }
                }
        }
        PV ones;
        const typename O_::PE one = (typename O_::PE)__builtin_amdgcn_exp2f(-lift);
#pragma unroll
        for (int j = 0; j < 8; ++j) ones[j] = one;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int n = NP - 1; n >= 0; --n) l[rt] = mfma(ones, pf[rt][k][n], l[rt]);
    }

    __device__ __forceinline__ float unit() const { return __builtin_amdgcn_exp2f(e_ref - ROOM); }

    // results, or this chunk's part of them
    __device__ __forceinline__ void finish(const AttendParams &p, const Unit &u, int c0, int c1, int h,
                                           int split, bool any) {
        const int lane = lane_id(), col = lane & 15, g = lane >> 4;
        const float un = unit();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int c = c0 + rt * 16 + col;
            if (c >= c1) continue;
            const int t = u.t0 + c / p.rep, hq = h * p.rep + c % p.rep;
            const float sum = l[rt][0];
            if (p.S == 1) {
                T *row = (T *)p.out + t * p.o_st + hq * p.o_sh;
                const float f = sum == 0.f ? 0.f : un / sum;
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    const int x = i * 16 + 4 * g;
                    T v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        Cvt<T>::store(v + r, sum == 0.f ? 0.f : o[rt][i][r] * f);
                    if (p.o_vec) {
                        if (x < p.d)
                            __builtin_memcpy(__builtin_assume_aligned(row + x, 4 * sizeof(T)), v,
                                             sizeof(v));
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (x + r < p.d) row[x + r] = v[r];
                    }
                }
            } else {
                const int64_t at = ((int64_t)t * p.Hq + hq) * p.s_stride + split;
                if (any) {
#pragma unroll
                    for (int i = 0; i < ND; ++i)
                        *(f32x4 *)(p.part_o + at * D + i * 16 + 4 * g) = o[rt][i] * un;
                }
                if (g == 0) {
                    p.part_ml[2 * at] = m[rt];
                    p.part_ml[2 * at + 1] = sum;
                }
            }
        }
    }
};

// launches of ssa_cache_prompt.hip: requests with more columns than `many`
int ssa_cache_prompt_max_rt(int dtype, int D);          // most 16-column tiles a wave takes
void ssa_cache_prompt_launch(const AttendParams &p, int dtype, int D, int KT, int RT, hipStream_t st);
