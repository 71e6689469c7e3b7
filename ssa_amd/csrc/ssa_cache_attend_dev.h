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
    UNITS_FEW,      // one for each request with at most `many` columns (CT >= many)
    UNITS_MANY,     // those of the others
};

struct AttendParams {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *starts, *requests, *positions, *pages;
    const void *q;
    void *out;
    float *part_ml, *part_o;                  // (columns, S, 2), (columns, S, D)
    int64_t num_pages, table_stride, q_st, q_sh, o_st, o_sh;
    int32_t T, R, width, Hq, Hkv, rep, d, page_shift, top, S, chunk, mode, many, units;
    int32_t q_vec, o_vec;                     // rows of q in 16-byte pieces, of out in 4 elements
    float scale;                              // softmax scale * log2(e)
};

struct Unit {
    int req, t0, c0, c1;    // row t0 + c / rep, head c % rep, for c in [c0, c1)
    int u;
};

// Where the chunks of a column are: by row and head; in UNITS_FEW, whose requests are
// cut into more chunks than all rows have room for, by unit and column.
__device__ __forceinline__ int64_t part_of(const AttendParams &p, const Unit &x, int c, int h) {
    if (p.mode == UNITS_FEW) return (((int64_t)x.u * p.Hkv + h) * p.many + c) * p.S;
    const int t = x.t0 + c / p.rep;
    return ((int64_t)t * p.Hq + h * p.rep + c % p.rep) * p.S;
}

// The columns of unit u, false if there are none.  Requests' units are numbered
// without a list: in UNITS_ALL and UNITS_MANY request r (R stands for the rows
// behind the last one) has its units from floor(starts[r] rep / CT) + r on, which
// leaves each request ceil(rows rep / CT); found by binary search.
__device__ __forceinline__ bool locate_unit(const AttendParams &p, int u, int CT, Unit &x) {
    x.u = u;
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
            lo = u;                           // CT >= many: one a request
            j = 0;
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
//    2^e_v into its addend: O is kept in units of 2^e_ref and p_j 2^lift, lift = e_v -
//    e_ref, is what multiplies the unscaled codes;
//  * sums of p come from the matrix unit, as one more row of V^T (the power of two
//    that undoes these units, so that they are the sums of p as rounded);
//  * O is rescaled only when a column's maximum has grown by more than 2^4, or lift
//    has left 0 .. 6.  With 2^5 to spare below, p 2^(lift + 5) as an f16 stays under
//    2^15 and its rounding at 11 bits, or 2^-30 of the largest p.  Values more than
//    2^64 below the request's largest (of a page of zeros, as a rule, which has the
//    smallest scale there is) are taken as zeros: O in their units could leave fp32.
// For fp32 queries p is three bf16 terms (24 bits; V scaled, as bf16 holds every
// scale).
template <typename T, int D, int KT>
struct Columns {
    typedef Ops<T> O_;
    typedef typename O_::Q QV;
    typedef typename O_::P PV;
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int NQ = O_::NQ, NP = O_::NP;
    static constexpr int NB = KT / 16, DP = D / 64, ND = D / 16, KS = KT / 32;
    // p is kept 2^ROOM larger, O in units of 2^(e_ref - ROOM)
    static constexpr int ROOM = F32 ? 0 : 5, LIFT = 6;
    static constexpr float GROWN = 4.f;

    QV q[DP * 2][NQ];
    f32x4 o[ND], l;
    float m, scale;
    int e_ref, e_top;            // O's unit; the largest it has been
    int pos;                     // last key a column sees; none for it to lose if it is dead
    int most, least;             // of the live columns

    // columns c0 + lane % 16 below c1 of unit u, kv head h
    __device__ __forceinline__ void start(const AttendParams &p, const Unit &u, int c0, int c1, int h) {
        const int lane = lane_id(), col = lane & 15, g = lane >> 4;
        const bool neg = p.scale < 0.f;
        scale = fabsf(p.scale);
        e_ref = e_top = -10000;  // anything is larger, and O is 0
        most = -1;
        least = 0x7fffffff;
        const int c = c0 + col;
        const bool live = c < c1;
        // dead lanes load the last live column, so that no load waits for another
        const int cc = min(c, c1 - 1), t = u.t0 + cc / p.rep;
        const int32_t req = p.requests[t], at = p.positions[t];
        const int seen = live && u.req >= 0 && req == u.req ? at : -1;
        most = max(most, seen);
        if (live) least = min(least, seen);
        pos = live ? seen : 0x7fffffff;
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
                    q[s][n][j] = b;
                    v -= (float)b;
                }
            }
        m = -INFINITY;
        l = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        most = (int)wave_max_u((uint32_t)(most + 1)) - 1;
        most = min(most, (p.width << p.page_shift) - 1);
        least = (int)wave_min_u((uint32_t)(least + 1)) - 1;
    }

    // scores to probabilities: key scale ks, value scale vs, first key of the tile;
    // l takes their sums.  False where the tile's values count as zeros.
    __device__ __forceinline__ bool softmax(f32x4 (&s)[NB], float ks, float vs, int key0,
                                            PV (&pf)[KS][NP]) {
        const int g = lane_id() >> 4;
        float c = scale * ks;                 // log2 units of a score's unit
        if (key0 + KT - 1 > least) {          // some column ends in this tile
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    s[b][r] = key0 + KT / 4 * g + 4 * b + r <= pos ? s[b][r] * c : -INFINITY;
            c = 1.f;
        }
        const int ev = F32 ? 0 : (int)(__builtin_amdgcn_readfirstlane(__float_as_uint(vs)) >> 23) - 127;
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[b][r]);
        mx *= c;
        const bool tiny = !F32 && ev < e_top - 64;
        const bool move = !tiny && (ev > e_ref + LIFT || ev < e_ref);
        if (wave_ballot(mx > m + GROWN) || move) {
            const int e_new = move ? (F32 ? 0 : ev - 3) : e_ref;
            const float unit = __builtin_amdgcn_exp2f((float)(e_ref - e_new));
            e_ref = e_new;
            e_top = max(e_top, e_new);
            float v = fmaxf(mx, __shfl_xor(mx, 16, SSA_WAVE));
            v = fmaxf(v, __shfl_xor(v, 32, SSA_WAVE));
            v = fmaxf(v, m);
            const float a = __builtin_amdgcn_exp2f(m - (v == -INFINITY ? 0.f : v));
            m = v;
            l *= a;
            const float au = a * unit;
#pragma unroll
            for (int i = 0; i < ND; ++i) o[i] *= au;
        }
        const float lift = (float)(tiny ? ROOM : ev - e_ref + ROOM);
        const float sub = lift - (m == -INFINITY ? 0.f : m);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = __builtin_amdgcn_exp2f(fmaf(s[b][r], c, sub));
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    const typename O_::PE e = (typename O_::PE)v;
                    pf[b >> 1][n][(b & 1) * 4 + r] = e;
                    if (n + 1 < NP) v -= (float)e;
                }
            }
        PV ones;
        const typename O_::PE one = (typename O_::PE)__builtin_amdgcn_exp2f(-lift);
#pragma unroll
        for (int j = 0; j < 8; ++j) ones[j] = one;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int n = NP - 1; n >= 0; --n) l = mfma(ones, pf[k][n], l);
        return !tiny;
    }

    __device__ __forceinline__ float unit() const { return __builtin_amdgcn_exp2f((float)(e_ref - ROOM)); }

    // results, or this chunk's part of them
    __device__ __forceinline__ void finish(const AttendParams &p, const Unit &u, int c0, int c1, int h,
                                           int split, bool any) {
        const int lane = lane_id(), col = lane & 15, g = lane >> 4;
        const float un = unit();
        const int c = c0 + col;
        if (c >= c1) return;
        const int t = u.t0 + c / p.rep, hq = h * p.rep + c % p.rep;
        const float sum = l[0];
        if (p.S == 1) {
            T *row = (T *)p.out + t * p.o_st + hq * p.o_sh;
            const float f = sum == 0.f ? 0.f : un / sum;
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                const int x = i * 16 + 4 * g;
                T v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    Cvt<T>::store(v + r, sum == 0.f ? 0.f : o[i][r] * f);
                if (p.o_vec) {
                    if (x < p.d)
                        __builtin_memcpy(__builtin_assume_aligned(row + x, 4 * sizeof(T)), v, sizeof(v));
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (x + r < p.d) row[x + r] = v[r];
                }
            }
        } else {
            const int64_t at = part_of(p, u, c, h) + split;
            if (any) {
#pragma unroll
                for (int i = 0; i < ND; ++i)
                    *(f32x4 *)(p.part_o + at * D + i * 16 + 4 * g) = o[i] * un;
            }
            if (g == 0) {
                p.part_ml[2 * at] = m;
                p.part_ml[2 * at + 1] = sum;
            }
        }
    }
};

// 16-byte pieces of LDS that attend_unit uses
template <int D, int KT, bool SHARED>
constexpr int attend_lds() {
    const int moving = ATT_WAVES * KT * D / 16, joined = SHARED ? 16 * (D + 4) / 4 : 0;
    return (moving > joined ? moving : joined) + ATT_WAVES * 16 / 2;
}

// A unit is 16 columns.  SHARED: a workgroup takes one unit and a chunk of its key
// tiles, its waves every fourth tile, and their sums are joined in LDS.  Otherwise
// each wave takes a unit of its own and all of its tiles, and nothing is joined.  A
// wave holds one tile's values and the next one's keys in flight, and looks page ids
// up a tile ahead of those.  (Units of 32 columns, for more than 16 query heads of a
// kv head, read their keys once and not twice, but a wave then holds twice the state
// and waits more: 64 tokens of 32 heads over one, 4k to 8k keys, 101 us to 65 us.)
template <typename T, int D, int KT, bool SHARED>
__device__ __forceinline__ void attend_unit(const AttendParams &p, unsigned block, int split,
                                            u32x4 *lds) {
    typedef Columns<T, D, KT> C;
    typedef typename C::PV PV;
    constexpr int NQ = C::NQ, NP = C::NP, NB = C::NB, DP = C::DP, ND = C::ND, KS = C::KS;
    constexpr int CT = 16, OS = D + 4;        // OS: row stride of the joined sums
    // each wave's pieces on their way to other lanes; then the joined sums
    u32x4 *x_lds = lds;
    constexpr int XW = KT * D / 16;
    float *o_lds = (float *)lds;
    float (*m_lds)[CT] = (float (*)[CT])(lds + attend_lds<D, KT, SHARED>() - ATT_WAVES * CT / 2);
    float (*l_lds)[CT] = m_lds + ATT_WAVES;

    const int lane = lane_id(), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    // kv heads run fastest: an XCD's workgroups share their heads' pages in its L2
    const int h = (int)(block % (unsigned)p.Hkv);
    int u = (int)(block / (unsigned)p.Hkv);
    if (!SHARED) u = u * ATT_WAVES + wave;
    Unit un;
    if (u >= p.units || !locate_unit(p, u, CT, un)) return;
    C w;
    w.start(p, un, un.c0, un.c1, h);

    const int page = 1 << p.page_shift, sub_shift = p.page_shift - (KT == 64 ? 6 : 5);
    const int32_t *list = p.pages ? p.pages + ((int64_t)un.t0 * p.Hkv + h) * p.top : nullptr;
    const int32_t *table = p.table + (int64_t)(un.req < 0 ? 0 : un.req) * p.table_stride;
    const int n_tiles = w.most < 0 ? 0 : (list ? p.top << sub_shift : w.most / KT + 1);
    const int tile0 = split * p.chunk, tile1 = min(tile0 + p.chunk, n_tiles);
    constexpr int STEP = SHARED ? ATT_WAVES : 1;

    // The logical page of a tile and its entry in the table, looked up a tile ahead
    // of its keys: the loads are unconditional (of some entry that is there) and
    // what they say is judged only where it is needed, so nothing waits for them.
    const int last_entry = (max(tile1, 1) - 1) >> sub_shift;
    auto look_up = [&](int tile) { return list ? list[min(tile >> sub_shift, last_entry)] : tile >> sub_shift; };
    auto entry = [&](int lp) { return table[max(0, min(lp, p.width - 1))]; };
    // the page's place in the cache, -1 if it is absent or unseen
    auto place = [&](int tile, int lp, int pg) {
        const int key0 = (lp << p.page_shift) + (tile & ((1 << sub_shift) - 1)) * KT;
        return tile < tile1 && lp >= 0 && lp < p.width && key0 <= w.most && pg >= 0 && pg < p.num_pages
                   ? pg : -1;
    };
    u32x4 *xk = x_lds + wave * XW;            // [block][64 columns][slot]
    u32x2 *xv = (u32x2 *)xk;                  // pages of 32: [16 columns][slot]
    const int lrow = lane >> 2, lpiece = lane & 3, to = slot_of(lrow, lpiece), from = slot_of(col, g);
    u32x4 kr[NB][DP];
    float ks = 0.f, vs = 0.f;
    auto fetch_keys = [&](int tile, int pg) {
        if (pg < 0) return;
        const int64_t ph = (int64_t)pg * p.Hkv + h;
        ks = p.ks[ph];
        vs = p.vs[ph];
        const uint8_t *kb = p.k + ph * page * D + (int64_t)(tile & ((1 << sub_shift) - 1)) * KT * D;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < DP; ++i)
                kr[b][i] = *(const u32x4 *)(kb + (KT / 4 * (lrow >> 2) + 4 * b + (lrow & 3)) * D + i * 64 + lpiece * 16);
    };

    int tile = tile0 + (SHARED ? wave : 0);
    int lp = 0, lp1 = 0, pg = -1;
    if (tile < tile1) {
        lp = look_up(tile);
        lp1 = look_up(tile + STEP);
        pg = place(tile, lp, entry(lp));
        fetch_keys(tile, pg);
    }
    for (; tile < tile1; tile += STEP) {
        int pg1, lp2;
        if (pg >= 0) {
            const int sub = tile & ((1 << sub_shift) - 1);
            const float kscale = ks, vscale = vs;
            const uint8_t *vb = p.v + ((int64_t)pg * p.Hkv + h) * D * page + sub * KT;
            uint32_t vr[ND][KT / 16];
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                const uint8_t *at = vb + ((i * 16 + lrow) << p.page_shift) + KT / 4 * lpiece;
                if constexpr (KT == 64) {
                    const u32x4 x = *(const u32x4 *)at;
                    vr[i][0] = x.x; vr[i][1] = x.y; vr[i][2] = x.z; vr[i][3] = x.w;
                } else {
                    const u32x2 x = *(const u32x2 *)at;
                    vr[i][0] = x.x; vr[i][1] = x.y;
                }
            }
            // loads go out in this order: values, then what the next tile's need
            __builtin_amdgcn_sched_barrier(0);
            const int entry1 = entry(lp1);
            lp2 = look_up(tile + 2 * STEP);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < DP; ++i) xk[(b * DP + i) * SSA_WAVE + to] = kr[b][i];
            wave_lds_sync();
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < DP; ++i) kr[b][i] = xk[(b * DP + i) * SSA_WAVE + from];
            __builtin_amdgcn_sched_barrier(0);
            f32x4 s[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < DP; ++i) {
                    const u32x4 x = kr[b][i];
                    const typename C::QV k0 = Ops<T>::key(x.x, x.y), k1 = Ops<T>::key(x.z, x.w);
#pragma unroll
                    for (int n = NQ - 1; n >= 0; --n) {
                        s[b] = mfma(k0, w.q[2 * i][n], s[b]);
                        s[b] = mfma(k1, w.q[2 * i + 1][n], s[b]);
                    }
                }
            }
            pg1 = place(tile + STEP, lp1, entry1);
            fetch_keys(tile + STEP, pg1);
            __builtin_amdgcn_sched_barrier(0);
            PV pf[KS][NP];
            const bool some = w.softmax(s, kscale, vscale, (lp << p.page_shift) + sub * KT, pf);
            wave_lds_sync();
            if (some) {
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    if constexpr (KT == 64)
                        xk[i * SSA_WAVE + to] = u32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]};
                    else
                        xv[i * SSA_WAVE + to] = u32x2{vr[i][0], vr[i][1]};
                }
                wave_lds_sync();
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    if constexpr (KT == 64) {
                        const u32x4 x = xk[i * SSA_WAVE + from];
                        vr[i][0] = x.x; vr[i][1] = x.y; vr[i][2] = x.z; vr[i][3] = x.w;
                    } else {
                        const u32x2 x = xv[i * SSA_WAVE + from];
                        vr[i][0] = x.x; vr[i][1] = x.y;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const PV vf = Ops<T>::value(vr[i][2 * k], vr[i][2 * k + 1], vscale);
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n)
                            w.o[i] = mfma(vf, pf[k][n], w.o[i]);
                    }
            }
            wave_lds_sync();
        } else {
            lp2 = look_up(tile + 2 * STEP);
            pg1 = place(tile + STEP, lp1, entry(lp1));
            fetch_keys(tile + STEP, pg1);
        }
        lp = lp1;
        pg = pg1;
        lp1 = lp2;
    }
    if constexpr (!SHARED) {
        w.finish(p, un, un.c0, un.c1, h, split, tile0 < tile1);
        return;
    }

    // join the waves: m, l, O in the waves' order
    if (g == 0) {
        m_lds[wave][col] = w.m;
        l_lds[wave][col] = w.l[0];
    }
    __syncthreads();                          // (and no wave's pieces are read any more)
    const float unit = w.unit();
    for (int v = 0; v < ATT_WAVES; ++v) {
        if (v == wave) {
            float mx = -INFINITY;
            for (int i = 0; i < ATT_WAVES; ++i) mx = fmaxf(mx, m_lds[i][col]);
            const float a = __builtin_amdgcn_exp2f(w.m - (mx == -INFINITY ? 0.f : mx)) * unit;
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                f32x4 *at = (f32x4 *)&o_lds[col * OS + i * 16 + 4 * g];
                const f32x4 x = w.o[i] * a;
                *at = v == 0 ? x : *at + x;
            }
        }
        __syncthreads();
    }
    for (int i = (int)threadIdx.x; i < CT * D; i += ATT_WAVES * SSA_WAVE) {
        const int c = i / D, x = i - c * D;
        if (un.c0 + c >= un.c1) break;
        float mx = -INFINITY, sum = 0.f;
        for (int v = 0; v < ATT_WAVES; ++v) mx = fmaxf(mx, m_lds[v][c]);
        const float ms = mx == -INFINITY ? 0.f : mx;
        for (int v = 0; v < ATT_WAVES; ++v)
            sum += l_lds[v][c] * __builtin_amdgcn_exp2f(m_lds[v][c] - ms);
        const int t = un.t0 + (un.c0 + c) / p.rep, hq = h * p.rep + (un.c0 + c) % p.rep;
        const float v = o_lds[c * OS + x];
        if (p.S == 1) {
            if (x < p.d)
                Cvt<T>::store((T *)p.out + t * p.o_st + hq * p.o_sh + x,
                              sum == 0.f ? 0.f : v / sum);
        } else {
            const int64_t at = part_of(p, un, un.c0 + c, h) + split;
            if (tile0 < tile1) p.part_o[at * D + x] = v;
            if (x == 0) {
                p.part_ml[2 * at] = mx;
                p.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// The kernel of ssa_cache_prompt.hip: p's units (requests with at most p.many columns)
// and q's (the others), ssa_cache_prompt_columns to a workgroup.
int ssa_cache_prompt_columns(int dtype, int D);
void ssa_cache_prompt_launch(const AttendParams &p, const AttendParams &q, int dtype, int D, int KT,
                             hipStream_t st);
