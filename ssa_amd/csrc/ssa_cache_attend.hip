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
#include "ssa_cache_dev.h"

namespace {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr int WAVES = 4;                      // of a workgroup
constexpr float LOG2E = 1.44269504088896340736f;

struct AttendParams {
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int32_t *table, *starts, *requests, *positions, *pages;
    const void *q;
    void *out;
    float *part_ml, *part_o;                  // (T * Hq, S, 2), (T * Hq, S, D)
    int64_t num_pages, table_stride, q_st, q_sh, o_st, o_sh;
    int32_t T, R, width, Hq, Hkv, rep, d, page_shift, top, S, chunk;
    float scale;                              // softmax scale * log2(e)
};

__device__ __forceinline__ bf16x8 zero8() {
    bf16x8 z;
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = (__bf16)0.f;
    return z;
}

// eight codes (two words) as bf16 times scale
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w0, uint32_t w1, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
    bf16x8 r;
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
    r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
    return r;
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// the request whose units hold unit u, where request r (R stands for the rows
// behind the last one) has its units from floor(starts[r] rep / CT) + r on: these
// leave each request ceil(rows rep / CT) and need no list
__device__ __forceinline__ int unit_request(const AttendParams &p, int u, int CT) {
    int lo = 0, hi = p.R;                     // last r with base(r) <= u
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        const int64_t base = (int64_t)p.starts[mid] * p.rep / CT + mid;
        if (base <= u) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A workgroup takes 16 RT columns (query rows of one request and kv head) and a
// chunk of the key tiles; its waves take every fourth tile of the chunk.
template <typename T, int D, int KT, int RT>
__global__ void __launch_bounds__(WAVES * SSA_WAVE)
cache_attend_kernel(AttendParams p) {
    constexpr int NQ = sizeof(T) == 4 ? 3 : (__is_same(T, f16_t) ? 2 : 1);
    constexpr int NP = sizeof(T) == 4 ? 3 : 2;
    constexpr int CT = 16 * RT, NB = KT / 16, DP = D / 64, ND = D / 16, KS = KT / 32;
    constexpr int OS = D + 4;                 // row stride of the waves' sums in LDS
    __shared__ float o_lds[CT * OS];
    __shared__ float m_lds[WAVES][CT], l_lds[WAVES][CT];

    const int lane = lane_id(), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    const int h = (int)blockIdx.y, split = (int)blockIdx.z;

    // this unit's columns: row t0 + c / rep, head c % rep, for c in [c0, c1)
    int req, t0, c0, c1;
    if (p.pages) {
        const int tiles = (p.rep + CT - 1) / CT;
        t0 = (int)blockIdx.x / tiles;
        c0 = ((int)blockIdx.x - t0 * tiles) * CT;
        c1 = min(c0 + CT, p.rep);
        req = p.requests[t0];
    } else {
        const int u = (int)blockIdx.x;
        const int r = unit_request(p, u, CT);
        t0 = p.starts[r];
        const int end = r < p.R ? p.starts[r + 1] : p.T;
        const int64_t j = u - ((int64_t)t0 * p.rep / CT + r);
        const int64_t cols = (int64_t)(min(end, p.T) - t0) * p.rep;
        if (t0 < 0 || j < 0 || j * CT >= cols) return;   // no such unit
        c0 = (int)(j * CT);
        c1 = (int)min((int64_t)c0 + CT, cols);
        req = r < p.R ? r : -1;
    }
    if (req >= p.R) req = -1;

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
            for (int n = 0; n < NQ; ++n) qf[rt][s][n] = zero8();
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
    for (int tile = tile0 + wave; tile < tile1; tile += WAVES) {
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
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mx = -INFINITY;
                for (int v = 0; v < WAVES; ++v) mx = fmaxf(mx, m_lds[v][rt * 16 + col]);
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
    for (int i = (int)threadIdx.x; i < CT * D; i += WAVES * SSA_WAVE) {
        const int c = i / D, x = i - c * D;
        if (c0 + c >= c1) break;
        float mx = -INFINITY, sum = 0.f;
        for (int v = 0; v < WAVES; ++v) mx = fmaxf(mx, m_lds[v][c]);
        const float ms = mx == -INFINITY ? 0.f : mx;
        for (int v = 0; v < WAVES; ++v)
            sum += l_lds[v][c] * __builtin_amdgcn_exp2f(m_lds[v][c] - ms);
        const int t = t0 + (c0 + c) / p.rep, hq = h * p.rep + (c0 + c) % p.rep;
        const float v = o_lds[c * OS + x];
        if (p.S == 1) {
            if (x < p.d)
                Cvt<T>::store((T *)p.out + t * p.o_st + hq * p.o_sh + x,
                              sum == 0.f ? 0.f : v / sum);
        } else {
            const int64_t at = ((int64_t)t * p.Hq + hq) * p.S + split;
            if (tile0 < tile1) p.part_o[at * D + x] = v;
            if (x == 0) {
                p.part_ml[2 * at] = mx;
                p.part_ml[2 * at + 1] = sum;
            }
        }
    }
}

// Joins the S chunks of each query row: one wave per row.  Bound by latency.
template <typename T, int D>
__global__ void __launch_bounds__(WAVES * SSA_WAVE)
cache_join_kernel(AttendParams p) {
    const int64_t row = (int64_t)blockIdx.x * WAVES + threadIdx.x / SSA_WAVE;
    if (row >= (int64_t)p.T * p.Hq) return;
    const int lane = lane_id();
    float mx = -INFINITY;
    for (int s = 0; s < p.S; ++s) mx = fmaxf(mx, p.part_ml[2 * (row * p.S + s)]);
    const float ms = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, o[D / 64];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) o[j] = 0.f;
    for (int s = 0; s < p.S; ++s) {
        const int64_t at = row * p.S + s;
        const float m = p.part_ml[2 * at], l = p.part_ml[2 * at + 1];
        if (l == 0.f) continue;               // nothing seen there (a NaN is not skipped)
        const float a = __builtin_amdgcn_exp2f(m - ms);
        sum += l * a;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) o[j] += p.part_o[at * D + j * 64 + lane] * a;
    }
    const int t = (int)(row / p.Hq), hq = (int)(row - (int64_t)t * p.Hq);
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        const int x = j * 64 + lane;
        if (x < p.d)
            Cvt<T>::store((T *)p.out + t * p.o_st + hq * p.o_sh + x, sum == 0.f ? 0.f : o[j] / sum);
    }
}

// What a call launches: columns per workgroup, workgroups over the columns, and
// the chunks that the key tiles are cut into.
struct AttendShape {
    int RT, KT, S, chunk;
    int64_t units;
};

AttendShape attend_shape(const ssa_cached_attention_args *a) {
    AttendShape s;
    const ssa_kv_cache &c = a->cache;
    const int rep = a->Hq / c.Hkv;
    s.KT = c.page < 64 ? 32 : 64;
    s.RT = rep > 16 ? 2 : 1;
    const int CT = 16 * s.RT;
    const int per_page = c.page / s.KT;
    int64_t tiles;                            // the most that a unit can have
    if (a->pages) {
        s.units = (int64_t)a->rows.T * ceil_div(rep, CT);
        tiles = (int64_t)a->top * per_page;
    } else {
        s.units = (int64_t)a->rows.T * rep / CT + a->rows.R + 1;
        tiles = (int64_t)a->rows.width * per_page;
    }
    // about 2,048 workgroups, with two tiles or more for each wave
    const int64_t want = ceil_div(2048, s.units * c.Hkv);
    int64_t chunk = ceil_div(tiles, want < 1 ? 1 : want);
    if (chunk < 2 * WAVES) chunk = 2 * WAVES;
    s.S = (int)ceil_div(tiles, chunk);
    if (s.S < 1) s.S = 1;
    s.chunk = (int)chunk;
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

template <typename T, int D, int KT, int RT>
void launch_attend(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    const dim3 grid((unsigned)s.units, (unsigned)p.Hkv, (unsigned)s.S);
    cache_attend_kernel<T, D, KT, RT><<<grid, WAVES * SSA_WAVE, 0, st>>>(p);
    if (s.S > 1)
        cache_join_kernel<T, D><<<(unsigned)ceil_div((int64_t)p.T * p.Hq, WAVES),
                                  WAVES * SSA_WAVE, 0, st>>>(p);
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
    if (s.S == 1) return 0;
    return (int64_t)a->rows.T * a->Hq * s.S * (2 + a->cache.D) * 4;
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
    SSA_CHECK_ARG(s.units < (1ll << 31) && s.S <= 65535, "cached_attention: too many rows");
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
    p.part_o = p.part_ml + (int64_t)a->rows.T * a->Hq * s.S * 2;
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
    p.chunk = s.chunk;
    p.scale = a->scale * LOG2E;
    const hipStream_t st = (hipStream_t)stream;
    if (a->dtype == SSA_F32) launch_attend_t<float>(p, s, c.D, st);
    else if (a->dtype == SSA_BF16) launch_attend_t<bf16_t>(p, s, c.D, st);
    else launch_attend_t<f16_t>(p, s, c.D, st);
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}
