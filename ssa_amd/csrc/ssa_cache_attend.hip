// ssa_cache_attend.hip -- attention over the paged 8-bit key/value cache.
//
// out = softmax(scale q K^T) V per query head, one pass over the keys with the
// running maximum m and sum l of the softmax:
//     m' = max(m, max_j s_j),  a = 2^(m - m'),  p_j = 2^(s_j - m'),
//     l' = a l + sum p_j,      O' = a O + p V     (s in units of log 2).
//
// Both products run on 16x16x32 bf16 MFMA, transposed: S^T = K Q^T and
// O^T = V^T P^T, so that a column is one query row throughout and the C layout of
// S^T is, lane for lane, the B layout of P^T.  That fixes which key a lane's rows
// stand for: in a tile of KT keys, row 4g + r of block b is key KT/4 g + 4b + r,
// and lane group g then reads KT/4 adjacent tokens of a transposed value row: 16
// (or 8) bytes, a wave 1 KB in one piece.  Key rows are read in 64-byte pieces.
// Nothing passes through LDS but the waves' results.
//
// Codes become bf16 with their scale in one instruction for two
// (v_cvt_scalef32_pk_bf16_fp8), exactly: a code has 4 significant bits and the
// scale is a power of two.  q and p are split into bf16 terms whose sum has the
// precision that is wanted (bf16 q 1 term, fp16 2, fp32 3; p 2 or 3), so every
// product is exact and only fp32 sums round.
#include "ssa_cache_attend_dev.h"

namespace {

// A workgroup takes 16 RT columns (query rows of one request and kv head) and a
// chunk of the key tiles; its waves take every fourth tile of the chunk.
template <typename T, int D, int KT, int RT>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE)
cache_attend_kernel(AttendParams p) {
    constexpr int NQ = sizeof(T) == 4 ? 3 : (__is_same(T, f16_t) ? 2 : 1);
    constexpr int NP = sizeof(T) == 4 ? 3 : 2;
    constexpr int CT = 16 * RT, NB = KT / 16, DP = D / 64, ND = D / 16, KS = KT / 32;
    constexpr int OS = D + 4;                 // row stride of the waves' sums in LDS
    __shared__ float o_lds[CT * OS];
    __shared__ float m_lds[ATT_WAVES][CT], l_lds[ATT_WAVES][CT];

    const int lane = lane_id(), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    const int h = (int)blockIdx.y, split = (int)blockIdx.z;

    Unit un;
    if (!locate_unit(p, (int)blockIdx.x, CT, un)) return;
    const int req = un.req, t0 = un.t0, c0 = un.c0, c1 = un.c1;

    int pos[RT];                              // last key each column sees
    int64_t qrow[RT];
    int most = -1;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int c = c0 + rt * 16 + col;
        const bool live = c < c1;
        const int t = t0 + c / p.rep;
        pos[rt] = live && req >= 0 && p.requests[t] == req ? p.positions[t] : -1;
        qrow[rt] = live ? t * p.q_st + (int64_t)(h * p.rep + c % p.rep) * p.q_sh : -1;
        most = max(most, pos[rt]);
    }
    most = __builtin_amdgcn_readfirstlane((int)wave_max_u((uint32_t)(most + 1))) - 1;
    const int page = 1 << p.page_shift;
    most = min(most, p.width * page - 1);

    const int sub_tiles = page / KT;          // 1, or 2 for pages of 128
    const int32_t *list = nullptr;
    int n_tiles = most < 0 ? 0 : most / KT + 1;
    if (p.pages) {
        list = p.pages + ((int64_t)t0 * p.Hkv + h) * p.top;
        n_tiles = most < 0 ? 0 : p.top * sub_tiles;
    }
    const int tile0 = split * p.chunk, tile1 = min(tile0 + p.chunk, n_tiles);

    bf16x8 qf[RT][DP * 2][NQ];
    f32x4 o[RT][ND];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.f;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < DP * 2; ++s)
#pragma unroll
            for (int n = 0; n < NQ; ++n) qf[rt][s][n] = bf16x8{};
    }
    if (tile0 < tile1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int s = 0; s < DP * 2; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int x = (s >> 1) * 64 + g * 16 + (s & 1) * 8 + j;
                    float v = qrow[rt] >= 0 && x < p.d ? to_f32(((const T *)p.q)[qrow[rt] + x]) : 0.f;
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        const __bf16 b = (__bf16)v;
                        qf[rt][s][n][j] = b;
                        v -= (float)b;
                    }
                }
    }

    const int32_t *table = p.table + (int64_t)(req < 0 ? 0 : req) * p.table_stride;
    for (int tile = tile0 + wave; tile < tile1; tile += ATT_WAVES) {
        int lp = tile / sub_tiles;
        const int sub = tile - lp * sub_tiles;
        if (list) lp = list[lp];
        if (lp < 0 || lp >= p.width) continue;
        const int pg = table[lp];
        if (pg < 0 || pg >= p.num_pages) continue;
        const int key0 = lp * page + sub * KT;
        if (key0 > most) continue;
        const int64_t ph = (int64_t)pg * p.Hkv + h;
        const float ks = p.ks[ph], vs = p.vs[ph];
        const uint8_t *kb = p.k + ph * page * D + (int64_t)sub * KT * D;
        const uint8_t *vb = p.v + ph * D * page + sub * KT;

        f32x4 s[RT][NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int key = KT / 4 * (col >> 2) + 4 * b + (col & 3);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DP; ++i) {
                const uint4 w = *(const uint4 *)(kb + key * D + i * 64 + g * 16);
                const bf16x8 k0 = codes_bf16(w.x, w.y, ks), k1 = codes_bf16(w.z, w.w, ks);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int n = NQ - 1; n >= 0; --n) {
                        s[rt][b] = mfma(k0, qf[rt][2 * i][n], s[rt][b]);
                        s[rt][b] = mfma(k1, qf[rt][2 * i + 1][n], s[rt][b]);
                    }
            }
        }
        bf16x8 pf[RT][KS][NP];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mx = m[rt];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = key0 + KT / 4 * g + 4 * b + r;
                    const float v = key <= pos[rt] ? s[rt][b][r] * p.scale : -INFINITY;
                    s[rt][b][r] = v;
                    mx = fmaxf(mx, v);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16, SSA_WAVE));
            mx = fmaxf(mx, __shfl_xor(mx, 32, SSA_WAVE));
            const float ms = mx == -INFINITY ? 0.f : mx;
            const float a = __builtin_amdgcn_exp2f(m[rt] - ms);
            m[rt] = mx;
            float sum = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = __builtin_amdgcn_exp2f(s[rt][b][r] - ms);
                    sum += v;
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const __bf16 t = (__bf16)v;
                        pf[rt][b >> 1][n][(b & 1) * 4 + r] = t;
                        v -= (float)t;
                    }
                }
            l[rt] = l[rt] * a + sum;
#pragma unroll
            for (int i = 0; i < ND; ++i) o[rt][i] *= a;
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            const uint8_t *at = vb + (int64_t)(i * 16 + col) * page + KT / 4 * g;
            uint32_t w[KT / 16];
            if constexpr (KT == 64) {
                const uint4 u = *(const uint4 *)at;
                w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            } else {
                const uint2 u = *(const uint2 *)at;
                w[0] = u.x; w[1] = u.y;
            }
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const bf16x8 vf = codes_bf16(w[2 * k], w[2 * k + 1], vs);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int n = NP - 1; n >= 0; --n) o[rt][i] = mfma(vf, pf[rt][k][n], o[rt][i]);
            }
        }
    }

    // join the waves: l over the lane groups, then m, l, O over the waves in order
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16, SSA_WAVE);
        l[rt] += __shfl_xor(l[rt], 32, SSA_WAVE);
        if (g == 0) {
            m_lds[wave][rt * 16 + col] = m[rt];
            l_lds[wave][rt * 16 + col] = l[rt];
        }
    }
    __syncthreads();
    for (int w = 0; w < ATT_WAVES; ++w) {
        if (w == wave) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mx = -INFINITY;
                for (int v = 0; v < ATT_WAVES; ++v) mx = fmaxf(mx, m_lds[v][rt * 16 + col]);
                const float a = __builtin_amdgcn_exp2f(m[rt] - (mx == -INFINITY ? 0.f : mx));
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    f32x4 *at = (f32x4 *)&o_lds[(rt * 16 + col) * OS + i * 16 + 4 * g];
                    const f32x4 x = o[rt][i] * a;
                    *at = w == 0 ? x : *at + x;
                }
            }
        }
        __syncthreads();
    }
    for (int i = (int)threadIdx.x; i < CT * D; i += ATT_WAVES * SSA_WAVE) {
        const int c = i / D, x = i - c * D;
        if (c0 + c >= c1) break;
        float mx = -INFINITY, sum = 0.f;
        for (int v = 0; v < ATT_WAVES; ++v) mx = fmaxf(mx, m_lds[v][c]);
        const float ms = mx == -INFINITY ? 0.f : mx;
        for (int v = 0; v < ATT_WAVES; ++v)
            sum += l_lds[v][c] * __builtin_amdgcn_exp2f(m_lds[v][c] - ms);
        const int t = t0 + (c0 + c) / p.rep, hq = h * p.rep + (c0 + c) % p.rep;
        const float v = o_lds[c * OS + x];
        if (p.S == 1) {
            if (x < p.d)
                Cvt<T>::store((T *)p.out + t * p.o_st + hq * p.o_sh + x,
                              sum == 0.f ? 0.f : v / sum);
        } else {
            const int64_t at = ((int64_t)t * p.Hq + hq) * p.s_stride + split;
            if (tile0 < tile1) p.part_o[at * D + x] = v;
            if (x == 0) {
                p.part_ml[2 * at] = mx;
                p.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// Joins the S chunks of each column: one wave per column.  Bound by latency, so the
// chunks' weights are formed side by side, a lane each.
template <typename T, int D>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE)
cache_join_kernel(AttendParams p, int CT) {
    Unit un;
    if (!locate_unit(p, (int)blockIdx.x, CT, un)) return;
    const int c = un.c0 + (int)blockIdx.z * ATT_WAVES + (int)threadIdx.x / SSA_WAVE;
    if (c >= un.c1) return;
    const int lane = lane_id();
    const int t = un.t0 + c / p.rep, hq = (int)blockIdx.y * p.rep + c % p.rep;
    const int64_t row = ((int64_t)t * p.Hq + hq) * p.s_stride;
    float mx = -INFINITY;
    for (int s = lane; s < p.S; s += SSA_WAVE) mx = fmaxf(mx, p.part_ml[2 * (row + s)]);
    mx = wave_max(mx);
    const float ms = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, o[D / 64];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) o[j] = 0.f;
    for (int s0 = 0; s0 < p.S; s0 += SSA_WAVE) {
        const int s = s0 + lane;
        float w = 0.f, l = 0.f;
        if (s < p.S) {
            l = p.part_ml[2 * (row + s) + 1];
            w = __builtin_amdgcn_exp2f(p.part_ml[2 * (row + s)] - ms);
        }
        sum += l * w;
        // a chunk that saw nothing (l = 0) has written no sums; a NaN is not skipped
        uint64_t some = wave_ballot(l != 0.f);
        while (some) {
            const int i = __ffsll((unsigned long long)some) - 1;
            some &= some - 1;
            const float wi = __shfl(w, i, SSA_WAVE);
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
                o[j] += p.part_o[(row + s0 + i) * D + j * 64 + lane] * wi;
        }
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        const int x = j * 64 + lane;
        if (x < p.d)
            Cvt<T>::store((T *)p.out + t * p.o_st + hq * p.o_sh + x, sum == 0.f ? 0.f : o[j] / sum);
    }
}

// What a call launches.  A request with more than MANY columns (rows times query
// heads of a kv head) shares its keys among that many matrix columns, enough for
// the kernel that stages key tiles in LDS (ssa_cache_prompt.hip); the others are
// bound by reading keys and go to the kernel above.  The lengths are on the GPU,
// so the host goes by T / R alone: at most 4 rows a request on average, all go
// one way (one launch); else both kernels are launched and each leaves the
// other's requests.
constexpr int MANY = 64;

struct AttendShape {
    int RT, KT, S, chunk;                     // of the kernel above
    int mode;
    int64_t units;
    bool prompt;
    int prompt_S, prompt_chunk, prompt_cols;
    int64_t prompt_units;
    int s_stride;
};

// chunks of the key tiles: about `wgs` workgroups in all, `least` tiles or more each
void split_tiles(int64_t tiles, int64_t units, int64_t wgs, int least, int *S, int *chunk) {
    const int64_t want = ceil_div(wgs, units);
    int64_t c = ceil_div(tiles, want < 1 ? 1 : want);
    if (c < least) c = least;
    *S = (int)ceil_div(tiles, c);
    if (*S < 1) *S = 1;
    *chunk = (int)c;
}

AttendShape attend_shape(const ssa_cached_attention_args *a) {
    AttendShape s = {};
    const ssa_kv_cache &c = a->cache;
    const int64_t T = a->rows.T, R = a->rows.R;
    const int rep = a->Hq / c.Hkv;
    s.KT = c.page < 64 ? 32 : 64;
    s.RT = rep > 16 ? 2 : 1;
    const int CT = 16 * s.RT;
    const int per_page = c.page / s.KT;
    int64_t tiles = (int64_t)a->rows.width * per_page;   // the most that a unit can have
    if (a->pages) {
        s.mode = UNITS_PAGES;
        s.units = T * ceil_div(rep, CT);
        tiles = (int64_t)a->top * per_page;
    } else if (T <= 4 * R || T * rep <= MANY) {
        s.mode = UNITS_ALL;
        s.units = T * rep / CT + R + 1;
    } else {
        s.mode = UNITS_FEW;
        s.units = (R + 1) * ceil_div(MANY, CT);
        s.prompt = true;
        s.prompt_cols = ssa_cache_prompt_columns(a->dtype, c.D);
        s.prompt_units = T * rep / s.prompt_cols + R + 1;
        split_tiles(tiles, s.prompt_units * c.Hkv, 512, 16, &s.prompt_S, &s.prompt_chunk);
    }
    // two tiles or more for each wave
    split_tiles(tiles, s.units * c.Hkv, 2048, 2 * ATT_WAVES, &s.S, &s.chunk);
    s.s_stride = s.prompt && s.prompt_S > s.S ? s.prompt_S : s.S;
    return s;
}

int check_attend(const ssa_cached_attention_args *a) {
    SSA_CHECK_ARG(a, "cached_attention: null arguments");
    int rc = ssa_check_cache(&a->cache);
    if (rc != SSA_OK) return rc;
    rc = ssa_check_rows(&a->rows, &a->cache);
    if (rc != SSA_OK) return rc;
    SSA_CHECK_ARG(a->dtype == SSA_F32 || a->dtype == SSA_BF16 || a->dtype == SSA_F16,
                  "cached_attention: dtype %d", a->dtype);
    SSA_CHECK_ARG(a->Hq >= 1 && a->Hq % a->cache.Hkv == 0,
                  "cached_attention: %d query heads are not a multiple of %d kv heads", a->Hq,
                  a->cache.Hkv);
    SSA_CHECK_ARG(!a->pages || (a->top >= 1 && a->top <= (1 << 24)),
                  "cached_attention: %d pages a row", a->top);
    SSA_CHECK_ARG((int64_t)a->rows.T * a->Hq < (1ll << 31),
                  "cached_attention: %d rows of %d heads pass 2^31", a->rows.T, a->Hq);
    return SSA_OK;
}

template <typename T, int D>
void launch_join(AttendParams p, int CT, hipStream_t st) {
    if (p.S == 1) return;
    const dim3 grid((unsigned)p.units, (unsigned)p.Hkv, (unsigned)ceil_div(CT, ATT_WAVES));
    cache_join_kernel<T, D><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p, CT);
}

template <typename T, int D, int KT, int RT>
void launch_attend(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    const dim3 grid((unsigned)p.units, (unsigned)p.Hkv, (unsigned)p.S);
    cache_attend_kernel<T, D, KT, RT><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
    launch_join<T, D>(p, 16 * RT, st);
    if (s.prompt) {
        AttendParams pp = p;
        pp.mode = UNITS_MANY;
        pp.units = (int32_t)s.prompt_units;
        pp.S = s.prompt_S;
        pp.chunk = s.prompt_chunk;
        ssa_cache_prompt_launch(pp, sizeof(T) == 4 ? SSA_F32 : (__is_same(T, f16_t) ? SSA_F16 : SSA_BF16),
                                D, KT, st);
        launch_join<T, D>(pp, s.prompt_cols, st);
    }
}

template <typename T, int D>
void launch_attend_d(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    if (s.KT == 32) {
        if (s.RT == 1) launch_attend<T, D, 32, 1>(p, s, st);
        else launch_attend<T, D, 32, 2>(p, s, st);
    } else {
        if (s.RT == 1) launch_attend<T, D, 64, 1>(p, s, st);
        else launch_attend<T, D, 64, 2>(p, s, st);
    }
}

template <typename T>
void launch_attend_t(const AttendParams &p, const AttendShape &s, int D, hipStream_t st) {
    if (D == 64) launch_attend_d<T, 64>(p, s, st);
    else if (D == 128) launch_attend_d<T, 128>(p, s, st);
    else launch_attend_d<T, 256>(p, s, st);
}

}  // namespace

extern "C" int64_t ssa_cached_attention_workspace_bytes(const ssa_cached_attention_args *a) {
    const int rc = check_attend(a);
    if (rc != SSA_OK) return rc;
    if (a->rows.T == 0) return 0;
    const AttendShape s = attend_shape(a);
    if (s.s_stride == 1) return 0;
    return (int64_t)a->rows.T * a->Hq * s.s_stride * (2 + a->cache.D) * 4;
}

extern "C" int ssa_cached_attention(const ssa_cached_attention_args *a, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
    const int64_t need = ssa_cached_attention_workspace_bytes(a);
    if (need < 0) return (int)need;
    if (a->rows.T == 0) return SSA_OK;
    SSA_CHECK_ARG(a->q && a->out, "cached_attention: null pointer");
    if (workspace_bytes < need || (need > 0 && !workspace)) {
        ssa_set_error("cached_attention: workspace of %lld bytes, %lld needed",
                      (long long)workspace_bytes, (long long)need);
        return SSA_E_WORKSPACE;
    }
    SSA_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "cached_attention: workspace alignment");
    const AttendShape s = attend_shape(a);
    SSA_CHECK_ARG(s.units < (1ll << 31) && s.S <= 65535 &&
                      s.prompt_units * a->cache.Hkv < (1ll << 31) && s.prompt_S <= 65535,
                  "cached_attention: too many rows");
    const ssa_kv_cache &c = a->cache;
    AttendParams p = {};
    p.k = (const uint8_t *)c.k_codes;
    p.v = (const uint8_t *)c.v_codes;
    p.ks = c.k_scale;
    p.vs = c.v_scale;
    p.table = a->rows.block_table;
    p.starts = a->rows.starts;
    p.requests = a->rows.requests;
    p.positions = a->rows.positions;
    p.pages = a->pages;
    p.q = a->q;
    p.out = a->out;
    p.part_ml = (float *)workspace;
    p.part_o = p.part_ml + (int64_t)a->rows.T * a->Hq * s.s_stride * 2;
    p.num_pages = c.num_pages;
    p.table_stride = a->rows.table_stride;
    p.q_st = a->q_st;
    p.q_sh = a->q_sh;
    p.o_st = a->o_st;
    p.o_sh = a->o_sh;
    p.T = a->rows.T;
    p.R = a->rows.R;
    p.width = a->rows.width;
    p.Hq = a->Hq;
    p.Hkv = c.Hkv;
    p.rep = a->Hq / c.Hkv;
    p.d = c.d;
    p.page_shift = c.page == 32 ? 5 : (c.page == 64 ? 6 : 7);
    p.top = a->top;
    p.S = s.S;
    p.s_stride = s.s_stride;
    p.mode = s.mode;
    p.many = MANY;
    p.units = (int32_t)s.units;
    p.chunk = s.chunk;
    p.scale = a->scale * LOG2E;
    const hipStream_t st = (hipStream_t)stream;
    if (a->dtype == SSA_F32) launch_attend_t<float>(p, s, c.D, st);
    else if (a->dtype == SSA_BF16) launch_attend_t<bf16_t>(p, s, c.D, st);
    else launch_attend_t<f16_t>(p, s, c.D, st);
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}
