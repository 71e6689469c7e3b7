// ssa_cache_prompt.hip -- attention over the paged 8-bit cache for many query rows
// of one request (prompts and their chunks).
//
// The products and the mapping of keys to lanes are those of ssa_cache_attend.hip
// (S^T = K Q^T, O^T = V^T P^T, a column is a query row, P^T stays in registers).
// Here each wave owns 16 RT columns and walks every key tile of the workgroup's
// range, so the tiles are shared: the waves convert a tile's codes to 16-bit floats
// once, into LDS, in the order in which the matrix operands read them (a fragment is
// 64 lanes x 16 bytes: every LDS access is a whole row of banks), double-buffered,
// with the next tile's codes already on their way from memory.  Bound by the matrix
// pipe and the exponentials together.
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
// scale).  Queries are exact: bf16, or f16, or three bf16 terms.
#include "ssa_cache_attend_dev.h"

namespace {

// V and Q as matrix operands, by the queries' type
template <typename T> struct Ops {                      // bf16
    typedef bf16x8 Q;
    typedef f16x8 P;
    static constexpr int NQ = 1, NP = 1;
    static __device__ __forceinline__ Q key(uint32_t a, uint32_t b) { return codes_bf16(a, b, 1.f); }
    static __device__ __forceinline__ P value(uint32_t a, uint32_t b, float) { return codes_f16(a, b); }
};
template <> struct Ops<f16_t> {
    typedef f16x8 Q;
    typedef f16x8 P;
    static constexpr int NQ = 1, NP = 1;
    static __device__ __forceinline__ Q key(uint32_t a, uint32_t b) { return codes_f16(a, b); }
    static __device__ __forceinline__ P value(uint32_t a, uint32_t b, float) { return codes_f16(a, b); }
};
template <> struct Ops<float> {
    typedef bf16x8 Q;
    typedef bf16x8 P;
    static constexpr int NQ = 3, NP = 3;
    static __device__ __forceinline__ Q key(uint32_t a, uint32_t b) { return codes_bf16(a, b, 1.f); }
    static __device__ __forceinline__ P value(uint32_t a, uint32_t b, float s) { return codes_bf16(a, b, s); }
};

template <typename V> struct Elem;
template <> struct Elem<bf16x8> { typedef __bf16 type; };
template <> struct Elem<f16x8> { typedef _Float16 type; };

template <typename T, int D, int KT, int RT>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE, D <= 128 ? 2 : 1)
cache_prompt_kernel(AttendParams p) {
    typedef Ops<T> O_;
    typedef typename O_::Q QV;
    typedef typename O_::P PV;
    typedef typename Elem<QV>::type QE;
    typedef typename Elem<PV>::type PE;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int NQ = O_::NQ, NP = O_::NP;
    constexpr int CT = ATT_WAVES * 16 * RT, NB = KT / 16, DP = D / 64, ND = D / 16, KS = KT / 32;
    // a load unit: 16 codes a lane, two fragments
    constexpr int KU = NB * DP, VU = ND * KS / 2, NU = KU + VU, UW = NU / ATT_WAVES;
    __shared__ uint4 frag[2][2 * NU][SSA_WAVE];
    __shared__ int most_lds[ATT_WAVES];

    const int lane = lane_id(), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    // kv heads run fastest: an XCD's workgroups share their heads' pages in its L2;
    // units run backwards, those with the most keys first
    const int h = (int)(blockIdx.x % (unsigned)p.Hkv);
    const int u = p.units - 1 - (int)(blockIdx.x / (unsigned)p.Hkv), split = (int)blockIdx.y;
    Unit un;
    if (!locate_unit(p, u, CT, un)) return;
    const int req = un.req;

    const int wc0 = un.c0 + wave * 16 * RT;   // this wave's first column
    int pos[RT];
    QV qf[RT][DP * 2][NQ];
    int most = -1, least = 0x7fffffff;
    const bool neg = p.scale < 0.f;
    const float scale = fabsf(p.scale);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int c = wc0 + rt * 16 + col;
        const bool live = c < un.c1;
        const int t = un.t0 + c / p.rep;
        const int seen = live && req >= 0 && p.requests[t] == req ? p.positions[t] : -1;
        most = max(most, seen);
        if (live) least = min(least, seen);
        pos[rt] = live ? seen : 0x7fffffff;   // dead columns need no mask of their own
        const T *row = (const T *)p.q + t * p.q_st + (int64_t)(h * p.rep + c % p.rep) * p.q_sh;
#pragma unroll
        for (int s = 0; s < DP * 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int x = (s >> 1) * 64 + g * 16 + (s & 1) * 8 + j;
                float v = live && x < p.d ? to_f32(row[x]) : 0.f;
                if (neg) v = -v;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const QE b = (QE)v;
                    qf[rt][s][n][j] = b;
                    v -= (float)b;
                }
            }
    }
    const int page = 1 << p.page_shift;
    most = (int)wave_max_u((uint32_t)(most + 1)) - 1;
    most = min(most, p.width * page - 1);
    least = (int)wave_min_u((uint32_t)(least + 1)) - 1;
    if (lane == 0) most_lds[wave] = most;
    __syncthreads();
    int most_wg = -1;
#pragma unroll
    for (int w = 0; w < ATT_WAVES; ++w) most_wg = max(most_wg, most_lds[w]);
    most_wg = __builtin_amdgcn_readfirstlane(most_wg);

    const int n_tiles = most_wg < 0 ? 0 : most_wg / KT + 1;
    const int tile0 = split * p.chunk, tile1 = min(tile0 + p.chunk, n_tiles);
    const int sub_shift = p.page_shift - (KT == 64 ? 6 : 5);
    const int32_t *table = p.table + (int64_t)(req < 0 ? 0 : req) * p.table_stride;

    // this wave's load units: key block b, columns 64 i.. ; or value rows
    int off[UW];
    uint4 raw[UW];
#pragma unroll
    for (int x = 0; x < UW; ++x) {
        const int un_ = wave * UW + x;
        if (un_ < KU) {
            const int b = un_ / DP, i = un_ % DP;
            off[x] = (KT / 4 * (col >> 2) + 4 * b + (col & 3)) * D + i * 64 + g * 16;
        } else {
            const int i = un_ - KU;
            off[x] = KT == 64 ? ((i * 16 + col) << p.page_shift) + 16 * g
                              : ((i * 32 + col) << p.page_shift) + 8 * g;
        }
    }
    struct Tile { int pg; float ks, vs; };
    // the page of a tile, -1 if it is absent
    auto page_of = [&](int tile) {
        if (tile >= tile1) return -1;
        const int pg = table[tile >> sub_shift];
        return pg >= 0 && pg < p.num_pages ? pg : -1;
    };
    auto fetch = [&](int tile, int pg, Tile &ti) {
        ti.pg = pg;
        if (pg < 0) return;
        const int sub = tile & ((1 << sub_shift) - 1);
        const int64_t ph = (int64_t)pg * p.Hkv + h;
        ti.ks = p.ks[ph];
        ti.vs = p.vs[ph];
        const uint8_t *kb = p.k + ph * D * page + sub * KT * D;
        const uint8_t *vb = p.v + ph * D * page + sub * KT;
#pragma unroll
        for (int x = 0; x < UW; ++x) {
            if (wave * UW + x < KU) {
                raw[x] = *(const uint4 *)(kb + off[x]);
            } else if (KT == 64) {
                raw[x] = *(const uint4 *)(vb + off[x]);
            } else {
                const uint2 a = *(const uint2 *)(vb + off[x]);
                const uint2 b = *(const uint2 *)(vb + off[x] + (16 << p.page_shift));
                raw[x] = uint4{a.x, a.y, b.x, b.y};
            }
        }
    };
    auto stage = [&](int buf, const Tile &ti) {
        if (ti.pg < 0) return;
#pragma unroll
        for (int x = 0; x < UW; ++x) {
            const int f = 2 * (wave * UW + x);
            if (wave * UW + x < KU) {
                *(QV *)&frag[buf][f][lane] = O_::key(raw[x].x, raw[x].y);
                *(QV *)&frag[buf][f + 1][lane] = O_::key(raw[x].z, raw[x].w);
            } else {
                *(PV *)&frag[buf][f][lane] = O_::value(raw[x].x, raw[x].y, ti.vs);
                *(PV *)&frag[buf][f + 1][lane] = O_::value(raw[x].z, raw[x].w, ti.vs);
            }
        }
    };

    f32x4 o[RT][ND], l[RT];
    float m[RT];
    // p is kept 2^ROOM larger, O in units of 2^(e_ref - ROOM)
    constexpr float ROOM = F32 ? 0.f : 5.f, GROWN = 4.f, LIFT = 6.f;
    float e_ref = 0.f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < ND; ++i) o[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    Tile cur{-1, 0.f, 0.f}, nxt{-1, 0.f, 0.f};
    int pg2 = -1;
    if (tile0 < tile1) {
        fetch(tile0, page_of(tile0), cur);
        stage(0, cur);
        fetch(tile0 + 1, page_of(tile0 + 1), nxt);
        pg2 = page_of(tile0 + 2);
    }
    __syncthreads();
    for (int tile = tile0; tile < tile1; ++tile) {
        const int buf = (tile - tile0) & 1;
        stage(buf ^ 1, nxt);
        Tile nn{-1, 0.f, 0.f};
        fetch(tile + 2, pg2, nn);
        pg2 = page_of(tile + 3);
        const int key0 = tile * KT;
        if (cur.pg >= 0 && key0 <= most) {
            f32x4 s[RT][NB];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int b = 0; b < NB; ++b) s[rt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < DP * 2; ++k) {
                    const QV kf = *(const QV *)&frag[buf][b * DP * 2 + k][lane];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int n = NQ - 1; n >= 0; --n) s[rt][b] = mfma(kf, qf[rt][k][n], s[rt][b]);
                }
            float c = scale * cur.ks;         // log2 units of a score's unit
            if (key0 + KT - 1 > least) {      // some column ends in this tile
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
            const float ev = F32 ? 0.f : (float)((int)(__float_as_uint(cur.vs) >> 23) - 127);
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
            PV pf[RT][KS][NP];
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
                            const PE e = (PE)v;
                            pf[rt][b >> 1][n][(b & 1) * 4 + r] = e;
                            if (n + 1 < NP) v -= (float)e;
                        }
                    }
            }
            PV ones;
#pragma unroll
            for (int j = 0; j < 8; ++j) ones[j] = (PE)__builtin_amdgcn_exp2f(-lift);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int n = NP - 1; n >= 0; --n) l[rt] = mfma(ones, pf[rt][k][n], l[rt]);
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const PV vf = *(const PV *)&frag[buf][2 * KU + i * KS + k][lane];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n) o[rt][i] = mfma(vf, pf[rt][k][n], o[rt][i]);
                }
        }
        __syncthreads();
        cur = nxt;
        nxt = nn;
    }

    const float unit = __builtin_amdgcn_exp2f(e_ref - ROOM);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int c = wc0 + rt * 16 + col;
        if (c >= un.c1) continue;
        const int t = un.t0 + c / p.rep, hq = h * p.rep + c % p.rep;
        const float sum = l[rt][0];
        if (p.S == 1) {
            T *row = (T *)p.out + t * p.o_st + hq * p.o_sh;
            const float f = sum == 0.f ? 0.f : unit / sum;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int x = i * 16 + 4 * g + r;
                    if (x < p.d) Cvt<T>::store(row + x, sum == 0.f ? 0.f : o[rt][i][r] * f);
                }
        } else {
            const int64_t at = ((int64_t)t * p.Hq + hq) * p.s_stride + split;
            if (tile0 < tile1) {
#pragma unroll
                for (int i = 0; i < ND; ++i)
                    *(f32x4 *)(p.part_o + at * D + i * 16 + 4 * g) = o[rt][i] * unit;
            }
            if (g == 0) {
                p.part_ml[2 * at] = m[rt];
                p.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// Columns per wave: as many as the registers hold beside O (RT D / 4), the scores
// and the queries.
template <typename T, int D> constexpr int prompt_rt() {
    return sizeof(T) == 4 ? (D <= 64 ? 2 : 1) : (D <= 64 ? 4 : 2);
}

template <typename T, int D>
void launch_d(const AttendParams &p, int KT, hipStream_t st) {
    constexpr int RT = prompt_rt<T, D>();
    const dim3 grid((unsigned)(p.units * p.Hkv), (unsigned)p.S);
    if (KT == 32) cache_prompt_kernel<T, D, 32, RT><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
    else cache_prompt_kernel<T, D, 64, RT><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
}

template <typename T>
void launch_t(const AttendParams &p, int D, int KT, hipStream_t st) {
    if (D == 64) launch_d<T, 64>(p, KT, st);
    else if (D == 128) launch_d<T, 128>(p, KT, st);
    else launch_d<T, 256>(p, KT, st);
}

}  // namespace

int ssa_cache_prompt_columns(int dtype, int D) {
    const int rt = dtype == SSA_F32
        ? (D == 64 ? prompt_rt<float, 64>() : D == 128 ? prompt_rt<float, 128>() : prompt_rt<float, 256>())
        : (D == 64 ? prompt_rt<bf16_t, 64>() : D == 128 ? prompt_rt<bf16_t, 128>()
                                                        : prompt_rt<bf16_t, 256>());
    return ATT_WAVES * 16 * rt;
}

void ssa_cache_prompt_launch(const AttendParams &p, int dtype, int D, int KT, hipStream_t st) {
    if (dtype == SSA_F32) launch_t<float>(p, D, KT, st);
    else if (dtype == SSA_BF16) launch_t<bf16_t>(p, D, KT, st);
    else launch_t<f16_t>(p, D, KT, st);
}
