// ssa_cache_attend.hip -- attention over the paged 8-bit key/value cache.
//
// out = softmax(scale q K^T) V per query head, one pass over the keys with the
// running maximum m and sum l of the softmax:
//     m' = max(m, max_j s_j),  a = 2^(m - m'),  p_j = 2^(s_j - m'),
//     l' = a l + sum p_j,      O' = a O + p V     (s in units of log 2).
//
// Both products run on 16x16x32 MFMA (K Q^T in bf16, for fp16 queries in f16; V^T P^T
// in f16, for fp32 queries in bf16), transposed: S^T = K Q^T and
// O^T = V^T P^T, so that a column is one query row throughout and the C layout of
// S^T is, lane for lane, the B layout of P^T.  That fixes which key a lane's rows
// stand for: in a tile of KT keys, row 4g + r of block b is key KT/4 g + 4b + r,
// and lane group g then reads KT/4 adjacent tokens of a transposed value row: 16
// (or 8) bytes, a wave 1 KB in one piece.  Key rows are read in 64-byte pieces.
//
// Codes become 16-bit floats in one instruction for two, exactly (a code has 4
// significant bits), and queries are exact too, so products are and only fp32 sums
// round; probabilities round to 11 bits, for fp32 queries to 24.
//
// Single tokens are bound by reading codes: 16 over 5k to 32k keys (32 / 8 heads, d
// 128, bf16) take 122 us, 4.7 TB/s, where a large copy reaches 4.8.  Chosen pages of a
// prompt's rows are bound by the L2, each row having a list of its own.
#include "ssa_cache_attend_dev.h"

namespace {

// A wave a unit fits three waves a SIMD (1,024 rows of 16 chosen pages: 134 us, with two
// 147 us); four waves to a unit are better with two and more in flight each (16 tokens,
// as above: 126 us, with three 151 us).
template <typename T, int D, int KT, bool SHARED>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE, D <= 128 ? (SHARED || sizeof(T) == 4 ? 2 : 3) : 1)
cache_attend_kernel(AttendParams p) {
    __shared__ u32x4 lds[attend_lds<D, KT, SHARED>()];
    attend_unit<T, D, KT, SHARED>(p, blockIdx.x, (int)blockIdx.y, lds);
}

// Joins the chunks of each column: D / 4 lanes a column, four channels each.  Bound by
// latency: the chunks' sums are read four at a time.  In a mixed call `q` describes
// the prompts' units, numbered behind p's.
template <typename T, int D>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE)
cache_join_kernel(AttendParams p, AttendParams q, int CT) {
    constexpr int LC = D / 4, PER = ATT_WAVES * SSA_WAVE / LC;
    const int x = (int)threadIdx.x % LC * 4;
    int64_t i = (int64_t)blockIdx.x * PER + (int)threadIdx.x / LC;
    int t, hq, S = p.S;
    const float *mls = p.part_ml, *pos = p.part_o;
    int64_t row;
    if (p.mode == UNITS_PAGES || p.mode == UNITS_ALL) {    // every row
        if (i >= (int64_t)p.T * p.Hq) return;
        t = (int)i / p.Hq;
        hq = (int)i - t * p.Hq;
        row = i * S;
    } else {
        // whole wavefronts look their unit up together: a wave's columns divide CT
        const int h = (int)blockIdx.y;
        const int64_t few = p.S > 1 ? (int64_t)p.units * CT : 0;
        const bool is_few = i < few;
        if (!is_few) {
            i -= few;
            S = q.S;
            mls = q.part_ml;
            pos = q.part_o;
        }
        const int u = (int)(i / CT);
        Unit un;
        if (is_few ? !locate_unit(p, u, CT, un)
                   : S == 1 || u >= q.units || !locate_unit(q, u, CT, un))
            return;
        const int c = un.c0 + (int)(i - (int64_t)u * CT);
        if (c >= un.c1) return;
        t = un.t0 + c / p.rep;
        hq = h * p.rep + c % p.rep;
        row = part_of(is_few ? p : q, un, c, h);
    }
    const float2 *ml = (const float2 *)mls + row;
    const float *po = pos + row * D + x;
    // the chunks' maxima and sums, a lane each, LC at a time
    const int lane = (int)threadIdx.x % LC;
    float mx = -INFINITY;
    for (int s = lane; s < S; s += LC) mx = fmaxf(mx, ml[s].x);
#pragma unroll
    for (int k = LC / 2; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, LC));
    const float ms = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    f32x4 o{0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < S; b += LC) {
        const float2 e = b + lane < S ? ml[b + lane] : float2{-INFINITY, 0.f};
        // a chunk that saw nothing (l = 0) has written no sums; a NaN is not skipped
        const float w = e.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(e.x - ms);
        sum += e.y == 0.f ? 0.f : e.y * w;
        const int n = min(LC, S - b);
        for (int s0 = 0; s0 < n; s0 += 4) {
            float wj[4];
            f32x4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                wj[j] = s0 + j < n ? __shfl(w, s0 + j, LC) : 0.f;
                v[j] = wj[j] == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f}
                                    : *(const f32x4 *)(po + (int64_t)(b + s0 + j) * D);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) o += v[j] * wj[j];
        }
    }
#pragma unroll
    for (int k = LC / 2; k > 0; k >>= 1) sum += __shfl_xor(sum, k, LC);
    T *out = (T *)p.out + t * p.o_st + hq * p.o_sh + x;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (x + j < p.d) Cvt<T>::store(out + j, sum == 0.f ? 0.f : o[j] / sum);
}

// What a call launches.  Many columns (rows times query heads of a kv head) of one
// request share its keys, staged in LDS (ssa_cache_prompt.hip); single tokens are
// bound by reading keys and go to the kernel above.  The lengths are on the GPU, so
// the host goes by T / R alone: at most 4 rows a request on average, all go one way
// (32 requests of 2 rows over up to 8k keys 97 us, the other way 118 us; 4 requests of
// 8 rows over up to 16k keys 59 us and 49 us; a prompt of 4,096 rows 514 us and 172
// us); else all the other, where requests with at most MANY columns are cut into chunks
// of their keys of their own, having few units each.
constexpr int MANY = 64;

struct AttendShape {
    int KT, mode, S, chunk;
    int64_t units;
    bool shared, prompt;
    int prompt_S, prompt_chunk, columns;      // columns: of a unit
    int64_t prompt_units;
    int64_t parts, prompt_parts;              // columns times chunks in the workspace
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
    s.columns = 16;
    s.shared = true;
    const int per_page = c.page / s.KT;
    int64_t tiles = (int64_t)a->rows.width * per_page;   // the most that a unit can have
    if (a->pages) {
        s.mode = UNITS_PAGES;
        s.units = T * ceil_div(rep, s.columns);
        tiles = (int64_t)a->top * per_page;
    } else if (T <= 4 * R || T * rep <= MANY) {
        s.mode = UNITS_ALL;
        s.units = T * rep / s.columns + R + 1;
    } else {
        s.mode = UNITS_FEW;
        s.columns = ssa_cache_prompt_columns(a->dtype, c.D);
        s.units = R + 1;
        s.prompt = true;
        s.prompt_units = T * rep / s.columns + R + 1;
        split_tiles(tiles, s.prompt_units * c.Hkv, 512, 4, &s.prompt_S, &s.prompt_chunk);
    }
    // Chunks of two tiles or more for each wave.  Lists of pages are equally long: as
    // many workgroups as the chip holds at once (512: 32 rows of 32 pages 34.7 us, with
    // 2,048 39.2 us).  Lengths are not: smaller chunks even them out (2,048: 16 tokens
    // over 5k to 32k keys 124 us, with 512 128 us, with 4,096 131 us).
    split_tiles(tiles, s.units * c.Hkv, a->pages ? 512 : 2048, 2 * ATT_WAVES, &s.S, &s.chunk);
    // A wave a unit, where there are units enough for that: over a few keys (256 tokens
    // over 4 pages of 64: 31 us, with four waves to a unit 43 us; over 24 pages 150 us
    // and 148 us), and where rows of one request, whose chosen pages are alike, run side
    // by side in a workgroup and read them from its CU's cache (512 rows of 24 pages 108
    // us, with four waves to a unit 139 us; 128 rows 48 us and 41 us).
    const int64_t waves = s.units * c.Hkv;
    if (!s.prompt && ((tiles * s.KT <= 512 && waves >= 1024) || (T > 4 * R && waves >= 2048))) {
        s.shared = false;
        s.S = 1;
        s.chunk = (int)(tiles < 0x7fffffff ? tiles : 0x7fffffff);
    }
    // no chunks, no parts; else about 2,048 workgroups' columns at most
    const int64_t few = s.prompt ? s.units * c.Hkv * MANY : T * a->Hq;
    s.parts = s.S > 1 ? few * s.S : 0;
    s.prompt_parts = s.prompt && s.prompt_S > 1 ? T * a->Hq * s.prompt_S : 0;
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

template <typename T, int D, int KT>
void launch_attend(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    if (s.shared) {
        const dim3 grid((unsigned)(p.units * p.Hkv), (unsigned)p.S);
        cache_attend_kernel<T, D, KT, true><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
    } else {
        const unsigned grid = (unsigned)(ceil_div(p.units, ATT_WAVES) * p.Hkv);
        cache_attend_kernel<T, D, KT, false><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p);
    }
}

template <typename T, int D>
void launch_join(const AttendParams &p, const AttendParams &q, const AttendShape &s, hipStream_t st) {
    if (p.S == 1 && (!s.prompt || q.S == 1)) return;
    constexpr int PER = ATT_WAVES * SSA_WAVE / (D / 4);
    const int64_t columns = !s.prompt ? (int64_t)p.T * p.Hq
                                      : ((p.S > 1 ? (int64_t)p.units : 0) +
                                         (q.S > 1 ? (int64_t)q.units : 0)) * s.columns;
    const dim3 grid((unsigned)ceil_div(columns, PER), s.prompt ? (unsigned)p.Hkv : 1u);
    cache_join_kernel<T, D><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p, q, s.columns);
}

template <typename T, int D>
void launch_attend_d(const AttendParams &p, const AttendShape &s, hipStream_t st) {
    AttendParams q = p;
    if (s.prompt) {
        q.mode = UNITS_MANY;
        q.units = (int32_t)s.prompt_units;
        q.S = s.prompt_S;
        q.chunk = s.prompt_chunk;
        q.part_ml = p.part_o + s.parts * D;
        q.part_o = q.part_ml + s.prompt_parts * 2;
        const int dtype = sizeof(T) == 4 ? SSA_F32 : (__is_same(T, f16_t) ? SSA_F16 : SSA_BF16);
        ssa_cache_prompt_launch(p, q, dtype, D, s.KT, st);
        return launch_join<T, D>(p, q, s, st);
    }
    if (s.KT == 32) launch_attend<T, D, 32>(p, s, st);
    else launch_attend<T, D, 64>(p, s, st);
    launch_join<T, D>(p, q, s, st);
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
    return (s.parts + s.prompt_parts) * (2 + a->cache.D) * 4;
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
    SSA_CHECK_ARG((s.units * s.S + s.prompt_units * s.prompt_S) * a->cache.Hkv < (1ll << 31) &&
                      s.S <= 65535,
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
    p.part_o = p.part_ml + s.parts * 2;
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
