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
//
// Codes become 16-bit floats in one instruction for two, exactly (a code has 4
// significant bits), and queries are exact too, so products are and only fp32 sums
// round; probabilities round to 11 bits, for fp32 queries to 24.
#include "ssa_cache_attend_dev.h"

namespace {

// A unit is 16 RT columns.  SHARED: a workgroup takes one unit and a chunk of its key
// tiles, its waves every fourth tile, and their sums are joined in LDS.  Otherwise
// each wave takes a unit of its own and all of its tiles: no joining, for calls with
// units enough to fill the chip.  A wave holds one tile's values and the next one's
// keys in flight, and looks page ids up a tile ahead of those.
template <typename T, int D, int KT, int RT, bool SHARED>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE, D <= 128 && RT == 1 ? 2 : 1)
cache_attend_kernel(AttendParams p) {
    typedef Columns<T, D, KT, RT> C;
    typedef typename C::PV PV;
    constexpr int NQ = C::NQ, NP = C::NP, NB = C::NB, DP = C::DP, ND = C::ND, KS = C::KS;
    constexpr int CT = 16 * RT, OS = D + 4;   // OS: row stride of the joined sums
    // each wave's pieces on their way to other lanes; then the joined sums
    constexpr int XW = KT * D / 16, XN = ATT_WAVES * XW, ON = SHARED ? CT * OS / 4 : 0;
    __shared__ u32x4 x_lds[XN > ON ? XN : ON];
    float *o_lds = (float *)x_lds;
    __shared__ float m_lds[ATT_WAVES][CT], l_lds[ATT_WAVES][CT];

    const int lane = lane_id(), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    // kv heads run fastest: an XCD's workgroups share their heads' pages in its L2
    const int h = (int)(blockIdx.x % (unsigned)p.Hkv), split = (int)blockIdx.y;
    int u = (int)(blockIdx.x / (unsigned)p.Hkv);
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
            f32x4 s[RT][NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < DP; ++i) {
                    const u32x4 x = xk[(b * DP + i) * SSA_WAVE + from];
                    const typename C::QV k0 = Ops<T>::key(x.x, x.y), k1 = Ops<T>::key(x.z, x.w);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int n = NQ - 1; n >= 0; --n) {
                            s[rt][b] = mfma(k0, w.q[rt][2 * i][n], s[rt][b]);
                            s[rt][b] = mfma(k1, w.q[rt][2 * i + 1][n], s[rt][b]);
                        }
                }
            }
            pg1 = place(tile + STEP, lp1, entry1);
            fetch_keys(tile + STEP, pg1);
            __builtin_amdgcn_sched_barrier(0);
            PV pf[RT][KS][NP];
            w.softmax(s, kscale, vscale, (lp << p.page_shift) + sub * KT, pf);
            wave_lds_sync();
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
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const PV vf = Ops<T>::value(vr[i][2 * k], vr[i][2 * k + 1], vscale);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n)
                            w.o[rt][i] = mfma(vf, pf[rt][k][n], w.o[rt][i]);
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
    if (g == 0)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m_lds[wave][rt * 16 + col] = w.m[rt];
            l_lds[wave][rt * 16 + col] = w.l[rt][0];
        }
    __syncthreads();                          // (and no wave's pieces are read any more)
    const float unit = w.unit();
    for (int v = 0; v < ATT_WAVES; ++v) {
        if (v == wave) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mx = -INFINITY;
                for (int i = 0; i < ATT_WAVES; ++i) mx = fmaxf(mx, m_lds[i][rt * 16 + col]);
                const float a = __builtin_amdgcn_exp2f(w.m[rt] - (mx == -INFINITY ? 0.f : mx)) * unit;
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    f32x4 *at = (f32x4 *)&o_lds[(rt * 16 + col) * OS + i * 16 + 4 * g];
                    const f32x4 x = w.o[rt][i] * a;
                    *at = v == 0 ? x : *at + x;
                }
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
    const int lane = lane_id();
    const int i = (int)blockIdx.x * ATT_WAVES + (int)threadIdx.x / SSA_WAVE;
    int t, hq;
    if (p.mode == UNITS_PAGES || p.mode == UNITS_ALL) {    // every row
        if (i >= p.T * p.Hq) return;
        t = i / p.Hq;
        hq = i - t * p.Hq;
    } else {
        Unit un;
        const int u = i / CT;
        if (u >= p.units || !locate_unit(p, u, CT, un)) return;
        const int c = un.c0 + i - u * CT;
        if (c >= un.c1) return;
        t = un.t0 + c / p.rep;
        hq = (int)blockIdx.y * p.rep + c % p.rep;
    }
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
    bool shared, prompt;
    int prompt_S, prompt_chunk, prompt_RT;
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
    // two tiles of heads share a wave's keys where the registers hold both
    s.RT = rep > 16 && c.D <= 128 ? 2 : 1;
    s.shared = true;
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
        // columns per wave: as many as leave two workgroups for every CU
        s.prompt_RT = ssa_cache_prompt_max_rt(a->dtype, c.D);
        for (;; s.prompt_RT /= 2) {
            s.prompt_units = T * rep / (ATT_WAVES * 16 * s.prompt_RT) + R + 1;
            if (s.prompt_RT == 1 || s.prompt_units * c.Hkv >= 512) break;
        }
        split_tiles(tiles, s.prompt_units * c.Hkv, 512, 4, &s.prompt_S, &s.prompt_chunk);
    }
    // two tiles or more for each wave
    split_tiles(tiles, s.units * c.Hkv, 2048, 2 * ATT_WAVES, &s.S, &s.chunk);
    if (!s.prompt && s.units * c.Hkv >= 4096) {
        s.shared = false;
        s.S = 1;
        s.chunk = (int)(tiles < 0x7fffffff ? tiles : 0x7fffffff);
    }
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
    const bool all = p.mode == UNITS_PAGES || p.mode == UNITS_ALL;
    const int64_t columns = all ? (int64_t)p.T * p.Hq : (int64_t)p.units * CT;
    const dim3 grid((unsigned)ceil_div(columns, ATT_WAVES), all ? 1u : (unsigned)p.Hkv);
    cache_join_kernel<T, D><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p, CT);
}

template <typename T, int D, int KT, int RT>
void launch_attend(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    if (s.shared) {
        const dim3 grid((unsigned)(p.units * p.Hkv), (unsigned)p.S);
        cache_attend_kernel<T, D, KT, RT, true><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
    } else {
        const unsigned grid = (unsigned)(ceil_div(p.units, ATT_WAVES) * p.Hkv);
        cache_attend_kernel<T, D, KT, RT, false><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
    }
    launch_join<T, D>(p, 16 * RT, st);
    if (s.prompt) {
        AttendParams pp = p;
        pp.mode = UNITS_MANY;
        pp.units = (int32_t)s.prompt_units;
        pp.S = s.prompt_S;
        pp.chunk = s.prompt_chunk;
        ssa_cache_prompt_launch(pp, sizeof(T) == 4 ? SSA_F32 : (__is_same(T, f16_t) ? SSA_F16 : SSA_BF16),
                                D, KT, s.prompt_RT, st);
        launch_join<T, D>(pp, ATT_WAVES * 16 * s.prompt_RT, st);
    }
}

template <typename T, int D>
void launch_attend_d(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    if constexpr (D <= 128)
        if (s.RT == 2) {
            if (s.KT == 32) launch_attend<T, D, 32, 2>(p, s, st);
            else launch_attend<T, D, 64, 2>(p, s, st);
            return;
        }
    if (s.KT == 32) launch_attend<T, D, 32, 1>(p, s, st);
    else launch_attend<T, D, 64, 1>(p, s, st);
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
    SSA_CHECK_ARG(s.units * a->cache.Hkv < (1ll << 31) && s.S <= 65535 &&
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
    const int es = a->dtype == SSA_F32 ? 4 : 2;
    p.q_vec = c.d % 8 == 0 && ((a->q_st | a->q_sh) * es) % 16 == 0 && ((uintptr_t)a->q & 15) == 0;
    p.o_vec = c.d % 4 == 0 && ((a->o_st | a->o_sh) * es) % (4 * es) == 0 &&
              ((uintptr_t)a->out & (4 * es - 1)) == 0;
    const hipStream_t st = (hipStream_t)stream;
    if (a->dtype == SSA_F32) launch_attend_t<float>(p, s, c.D, st);
    else if (a->dtype == SSA_BF16) launch_attend_t<bf16_t>(p, s, c.D, st);
    else launch_attend_t<f16_t>(p, s, c.D, st);
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}
