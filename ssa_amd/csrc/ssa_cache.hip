// ssa_cache.hip -- block tables, the append and the page selection of the paged
// 8-bit key/value cache (the attention over it is in ssa_cache_attend.hip).
#include "ssa_cache_dev.h"

namespace {

// ---------------------------------------------------------------------------- plan
// Everything follows from two prefix sums over the requests (their rows, and the
// pages they need), so every workgroup forms both in its LDS and then serves its
// share of the rows by binary search: one launch, no pass between workgroups.
// Bound by latency: two block scans and log2(R) LDS reads per row (8 requests 6.6 us,
// 1,000 with prompts among them 8.3 us).
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_MAX_R = 16384;      // two ints of LDS per request

// sums of lengths stop at 2^31 - 1, which no row index reaches
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) {
    const uint32_t s = a + b;
    return s > 0x7fffffffu ? 0x7fffffffu : s;
}

// exclusive saturating prefix sum over the workgroup, and the total
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *part, uint32_t *total) {
    const int lane = lane_id(), wave = (int)threadIdx.x / SSA_WAVE;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < SSA_WAVE; o <<= 1) {
        const uint32_t u = __shfl_up(inc, o, SSA_WAVE);
        if (lane >= o) inc = sat_add(inc, u);
    }
    __syncthreads();
    if (lane == SSA_WAVE - 1) part[wave] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / SSA_WAVE; ++w) {
        if (w < wave) before = sat_add(before, part[w]);
        all = sat_add(all, part[w]);
    }
    *total = all;
    const uint32_t own = __shfl_up(inc, 1, SSA_WAVE);
    return sat_add(before, lane == 0 ? 0u : own);
}

// PER: requests of a thread, held in registers between the scans
template <int PER>
__global__ void __launch_bounds__(PLAN_THREADS)
page_plan_kernel(ssa_page_plan_args a) {
    extern __shared__ uint32_t plan_lds[];
    __shared__ uint32_t part[PLAN_THREADS / SSA_WAVE];
    __shared__ uint32_t n_taken, n_refused;
    uint32_t *end = plan_lds;               // rows up to and with request r
    int32_t *base = (int32_t *)plan_lds + a.R;   // pages taken before r, -1 where refused
    const int r0 = (int)threadIdx.x * PER;
    const bool first_wg = blockIdx.x == 0;
    if (threadIdx.x == 0) n_taken = n_refused = 0;
    int c[PER], n[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {          // all in flight at once
        const int r = min(r0 + i, a.R - 1);
        c[i] = a.cached[r];
        n[i] = a.new_rows[r];
    }
    const uint32_t nfree = (uint32_t)max(0, min(*a.free_count, a.free_capacity));
    uint32_t sum = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (r0 + i < a.R) sum = sat_add(sum, (uint32_t)max(n[i], 0));
    uint32_t run = block_scan(sum, part, &total), need = 0;
    const int page_shift = 31 - __clz(a.page);
    int nd[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        nd[i] = -1;
        if (r0 + i >= a.R) continue;
        if (first_wg) a.starts[r0 + i] = (int32_t)run;
        run = sat_add(run, (uint32_t)max(n[i], 0));
        end[r0 + i] = run;
        const int64_t want = ((int64_t)c[i] + n[i] + a.page - 1) >> page_shift;
        const bool fits = c[i] >= 0 && n[i] >= 0 && want <= a.width && run <= (uint32_t)a.T;
        if (fits) nd[i] = (int)(want - (((int64_t)c[i] + a.page - 1) >> page_shift));
        need = sat_add(need, (uint32_t)max(nd[i], 0));
    }
    if (first_wg && threadIdx.x == 0) a.starts[a.R] = (int32_t)total;
    uint32_t upto = block_scan(need, part, &total);
    uint32_t taken = 0, refused = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (r0 + i >= a.R) continue;
        const uint32_t before = upto;
        upto = sat_add(upto, (uint32_t)max(nd[i], 0));
        const bool ok = nd[i] == 0 || (nd[i] > 0 && upto <= nfree);
        base[r0 + i] = ok ? (int32_t)min(before, nfree) : -1;
        taken += ok ? (uint32_t)nd[i] : 0u;
        refused += ok ? 0u : 1u;
        if (first_wg) a.lengths[r0 + i] = c[i] + (ok ? n[i] : 0);
    }
    __syncthreads();
    if (first_wg) {
        atomicAdd(&n_taken, taken);
        atomicAdd(&n_refused, refused);
        __syncthreads();
        if (threadIdx.x == 0) {
            *a.free_count_out = (int32_t)(nfree - n_taken);
            *a.refused = (int32_t)n_refused;
        }
    }
    for (int64_t t = (int64_t)blockIdx.x * PLAN_THREADS + threadIdx.x; t < a.T;
         t += (int64_t)gridDim.x * PLAN_THREADS) {
        int lo = 0, hi = a.R;                // first r with end[r] > t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (end[mid] > (uint32_t)t) hi = mid;
            else lo = mid + 1;
        }
        int64_t slot = -1;
        int32_t pos = -1, req = -1;
        if (lo < a.R && base[lo] >= 0) {
            const int held = a.cached[lo];
            req = lo;
            pos = held + (int32_t)(t - (lo ? end[lo - 1] : 0));
            const int col = pos >> page_shift, off = pos & (a.page - 1);
            const int had = (held + a.page - 1) >> page_shift;
            int32_t *entry = a.block_table + (int64_t)lo * a.table_stride + col;
            int32_t page;
            if (col < had) {
                page = *entry;
            } else {                         // a page taken now; its first row notes it
                page = a.free_pages[nfree - 1 - (uint32_t)(base[lo] + col - had)];
                if (off == 0) *entry = page;
            }
            slot = page < 0 ? -1 : (int64_t)page * a.page + off;
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
        a.requests[t] = req;
    }
}

template <int PER>
int launch_plan(const ssa_page_plan_args &a, hipStream_t s) {
    const size_t lds = (size_t)a.R * 8;
    SSA_ALLOW_LDS(page_plan_kernel<PER>, lds);
    // a thread a row: the scans are repeated side by side, rows would be in turn
    const int64_t want = ceil_div(a.T, PLAN_THREADS);
    const int grid = (int)(want < 1 ? 1 : (want > 1024 ? 1024 : want));
    page_plan_kernel<PER><<<grid, PLAN_THREADS, lds, s>>>(a);
    return SSA_OK;
}

// ---------------------------------------------------------------------------- append
// One workgroup per run of adjacent rows of one page and kv head: the run's
// largest magnitudes first (the page's scale has to hold before any code is
// rounded), then the codes, staged in LDS so that the transposed value codes go
// out 16 tokens at a time.  D / 8 lanes hold a row, 8 columns each, and keep it in
// registers between the two.  Bound by latency for single tokens (about five
// dependent steps: 64 tokens of 8 heads 6.6 us).  Prompts (8,193 rows of 8 heads, d
// 96 in fp16) take 23 us, 1.7 TB/s: bound by the wait for the rows, all of a
// workgroup's at once and two workgroups a CU (without forming codes 21 us).

// Eight adjacent columns of a row, in the registers they take as they are stored.
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
template <typename T> struct Row8 {                        // 16-bit types
    u32x4 w;
    __device__ __forceinline__ float get(int j) const {
        T t;
        t.x = (uint16_t)(w[j >> 1] >> 16 * (j & 1));
        return to_f32(t);
    }
    __device__ __forceinline__ void set(int j, T t) {
        w[j >> 1] = j & 1 ? (w[j >> 1] & 0xffffu) | (uint32_t)t.x << 16 : (uint32_t)t.x;
    }
    __device__ __forceinline__ void load(const T *p) { w = *(const u32x4 *)p; }
    __device__ __forceinline__ void cut(int n) {           // keeps the first n columns
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = n >= 2 * j + 2 ? w[j] : (n > 2 * j ? w[j] & 0xffffu : 0u);
    }
};
template <> struct Row8<float> {
    u32x4 w[2];
    __device__ __forceinline__ float get(int j) const { return __uint_as_float(w[j >> 2][j & 3]); }
    __device__ __forceinline__ void set(int j, float t) { w[j >> 2][j & 3] = __float_as_uint(t); }
    __device__ __forceinline__ void load(const float *p) {
        w[0] = *(const u32x4 *)p;
        w[1] = *(const u32x4 *)(p + 4);
    }
    __device__ __forceinline__ void cut(int n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2][j & 3] = n > j ? w[j >> 2][j & 3] : 0u;
    }
};

// columns x .. x + 7 of a row, anything past d.  VEC: d and the strides are multiples
// of 8 (the addresses of 16 bytes)
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const void *p, int64_t at, int x, int d, Row8<T> &v) {
    const T *q = (const T *)p + at;
    if (VEC) {
        v.load(q + (x < d ? x : 0));
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v.set(j, q[min(x + j, d - 1)]);
    }
}

// bits of the largest magnitude; a NaN's, its sign cleared, pass every number's
template <typename T>
__device__ __forceinline__ uint32_t max_bits8(const Row8<T> &v) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v.get(j)) & 0x7fffffffu);
    return m;
}
// the largest of N adjacent lanes' values (8, 16 or 32), in the vector unit: no lane
// permutation by way of the LDS, whose latency a row's steps would add up to
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    auto with = [&](int u) { v = max(v, (uint32_t)u); };
    with(__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true));      // lane ^ 1
    with(__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true));      // lane ^ 2
    with(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true));     // 7 - lane: the other four
    if (N >= 16) with(__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, true));   // 15 - lane
    if (N >= 32) with(__shfl_xor((int)v, 16, SSA_WAVE));
    return v;
}
template <typename T>
__device__ __forceinline__ uint2 codes8(const Row8<T> &v, float f) {
    return uint2{codes4(v.get(0) * f, v.get(1) * f, v.get(2) * f, v.get(3) * f),
                 codes4(v.get(4) * f, v.get(5) * f, v.get(6) * f, v.get(7) * f)};
}

// smallest e with a <= 448 * 2^e: 448 = 1.75 * 2^8
__device__ __forceinline__ int scale_exponent(float a) {
    const uint32_t u = __float_as_uint(a);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, SSA_CACHE_E_MIN), SSA_CACHE_E_MAX);
}
__device__ __forceinline__ float exp2_int(int e) {      // -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// a code's place in the order of the numbers (-126..126; NaN is told apart before)
__device__ __forceinline__ int code_rank(uint32_t code) {
    return (code & 0x80u) ? -(int)(code & 0x7fu) : (int)(code & 0x7fu);
}

template <typename T, int D, bool VEC, int APP_THREADS>
__global__ void __launch_bounds__(APP_THREADS, sizeof(T) == 4 || !VEC ? 2 : 3)
cache_append_kernel(ssa_cache_append_args a, int window) {
    constexpr int LPR = D / 8, RPW = APP_THREADS / LPR;   // lanes of a row, rows at a time
    constexpr int ROWS = 128 / RPW;                       // a thread's share of the most rows
    extern __shared__ uint4 app_lds[];
    __shared__ uint32_t kmax[128], vmax[128];     // bits of each row's largest magnitude
    __shared__ uint32_t page_max[2], any_bad;
    __shared__ int lo_lds[D], hi_lds[D];
    const ssa_kv_cache &c = a.cache;
    const int h = (int)blockIdx.y, ps = c.page, d = c.d, tid = (int)threadIdx.x;
    const int lane = lane_id(), rx = tid % LPR * 8, r0 = tid / LPR;
    const int64_t cap = c.num_pages * ps;
    uint8_t *kst = (uint8_t *)app_lds, *vst = kst + ps * D;      // [row][D] codes

    // the window's first rows of runs: every wave finds them for itself
    const int64_t w0 = (int64_t)blockIdx.x * window;
    int64_t at[3];                                // slots of rows w0 + lane, + 64, + 128
#pragma unroll
    for (int i = 0; i < 3; ++i) at[i] = w0 + 64 * i + lane < a.T ? a.slots[w0 + 64 * i + lane] : -1;
    const int64_t before = w0 > 0 ? a.slots[w0 - 1] : -1;
    const int64_t up = __shfl_up(at[0], 1, SSA_WAVE), prev = lane ? up : before;
    const int page_shift = 31 - __clz(ps);
    const bool first = lane < window && at[0] >= 0 && at[0] < cap &&
                       ((at[0] & (ps - 1)) == 0 || prev != at[0] - 1);
    uint64_t todo = wave_ballot(first);
    while (todo) {
        const int w = __ffsll((unsigned long long)todo) - 1;
        todo &= todo - 1;
        const int64_t t0 = w0 + w, slot = __shfl(at[0], w, SSA_WAVE);
        const int64_t pg = slot >> page_shift;
        const int off = (int)slot & (ps - 1);
        // length of the run: rows w0 + j at slot + j - w, within the page
        int n = ps - off;
#pragma unroll
        for (int i = 2; i >= 0; --i) {
            const int j = 64 * i + lane;
            const uint64_t m = wave_ballot(j > w && at[i] != slot + j - w);
            if (m) n = min(n, 64 * i + __ffsll((unsigned long long)m) - 1 - w);
        }
        const int64_t ph = pg * c.Hkv + h;
        const float k_old = off ? c.k_scale[ph] : 0.f, v_old = off ? c.v_scale[ph] : 0.f;
        const int64_t krow = t0 * a.k_st + (int64_t)h * a.k_sh;
        const int64_t vrow = t0 * a.v_st + (int64_t)h * a.v_sh;
        __syncthreads();                                   // the last run's LDS is read
        if (tid < 2) page_max[tid] = 0;
        if (tid == 2) any_bad = 0;
        Row8<T> kv[ROWS], vv[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = min(r0 + i * RPW, n - 1);        // past the run: its last row again
            if (i > 0 && i * RPW >= n) break;
            load_row8<T, VEC>(a.k, krow + r * a.k_st, rx, d, kv[i]);
            load_row8<T, VEC>(a.v, vrow + r * a.v_st, rx, d, vv[i]);
        }
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (i > 0 && i * RPW >= n) break;
            kv[i].cut(d - rx);         // here, so that no load above waits for another
            vv[i].cut(d - rx);
            const uint32_t km = lanes_max<LPR>(max_bits8(kv[i])), vm = lanes_max<LPR>(max_bits8(vv[i]));
            const int r = r0 + i * RPW;
            if (rx == 0 && r < n) {
                kmax[r] = km;
                vmax[r] = vm;
            }
        }
        __syncthreads();
        if (tid < n) {
            const uint32_t big = __float_as_uint(SSA_CACHE_TOO_BIG);
            if (kmax[tid] >= big || vmax[tid] >= big) {
                kmax[tid] = 0xffffffffu;                   // marks the row
                any_bad = 1;
            } else {
                atomicMax(&page_max[0], kmax[tid]);
                atomicMax(&page_max[1], vmax[tid]);
            }
        }
        __syncthreads();
        const float k_new = fmaxf(k_old, exp2_int(scale_exponent(__uint_as_float(page_max[0]))));
        const float v_new = fmaxf(v_old, exp2_int(scale_exponent(__uint_as_float(page_max[1]))));
        uint8_t *kp = (uint8_t *)c.k_codes + ph * ps * D, *vp = (uint8_t *)c.v_codes + ph * D * ps;
        uint8_t *bp = (uint8_t *)c.bounds + ph * 2 * D;
        if (k_old < k_new && off) {
            const float f = k_old / k_new;                 // both powers of two
            uint32_t *p = (uint32_t *)kp;
            for (int i = tid; i < off * D / 4; i += APP_THREADS) p[i] = codes4_scaled(p[i], f);
        }
        if (v_old < v_new && off) {
            const float f = v_old / v_new;
            uint32_t *p = (uint32_t *)vp;
            const int words = ps / 4;                      // of each channel's tokens
            for (int i = tid; i < D * words; i += APP_THREADS) {
                const int keep = off - 4 * (i & (words - 1));   // tokens below the run
                if (keep <= 0) continue;
                const uint32_t was = p[i], now = codes4_scaled(was, f);
                const uint32_t m = keep >= 4 ? ~0u : (1u << 8 * keep) - 1u;
                p[i] = (now & m) | (was & ~m);
            }
        }
        // bounds that stay, at the new scale
        const bool bad_page = any_bad != 0;
        for (int x = tid; x < D; x += APP_THREADS) {
            int lo = 127, hi = -127;
            if (off) {
                const float f = k_old / k_new;
                const uint32_t cd = codes2(code_f32<0>(bp[x]) * f, code_f32<0>(bp[D + x]) * f);
                const bool nan = (cd & 0x7fu) == SSA_CODE_NAN || ((cd >> 8) & 0x7fu) == SSA_CODE_NAN;
                lo = nan ? -127 : code_rank(cd & 0xffu);
                hi = nan ? 127 : code_rank(cd >> 8);
            }
            lo_lds[x] = lo;
            hi_lds[x] = hi;
        }
        const float ki = 1.f / k_new, vi = 1.f / v_new;    // exact
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int r = r0 + i * RPW;
            if (r >= n) break;
            uint2 kc = codes8(kv[i], ki), vc = codes8(vv[i], vi);
            if (kmax[r] == 0xffffffffu) {                  // a row that is not finite
                kc = uint2{SSA_CODE_NAN * 0x01010101u, SSA_CODE_NAN * 0x01010101u};
                vc = uint2{0, 0};
            }
            *(uint2 *)(kst + r * D + rx) = kc;
            *(uint2 *)(vst + r * D + rx) = vc;
            *(uint2 *)(kp + (int64_t)(off + r) * D + rx) = kc;
        }
        __syncthreads();
        // values: 4 columns x 16 tokens at a time, turned in registers
        const int g0 = off / 16, g1 = (off + n + 15) / 16;
        for (int i = tid; i < D / 4 * (g1 - g0); i += APP_THREADS) {
            const int x = i % (D / 4) * 4, tok = (g0 + i / (D / 4)) * 16;
            if (tok >= off && tok + 16 <= off + n) {
                uint32_t w[4][4];                          // [column][four tokens]
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t in[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        in[j] = *(const uint32_t *)(vst + (tok - off + 4 * q + j) * D + x);
                    // bytes (row, column) -> (column, row)
                    const uint32_t a0 = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u);
                    const uint32_t a1 = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
                    const uint32_t b0 = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
                    const uint32_t b1 = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
                    w[0][q] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
                    w[1][q] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
                    w[2][q] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
                    w[3][q] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *(uint4 *)(vp + (int64_t)(x + j) * ps + tok) =
                        uint4{w[j][0], w[j][1], w[j][2], w[j][3]};
            } else {
                const int e = min(tok + 16, off + n);
                for (int q = max(tok, off); q < e; ++q) {
                    const uint32_t v = *(const uint32_t *)(vst + (q - off) * D + x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) vp[(int64_t)(x + j) * ps + q] = (uint8_t)(v >> 8 * j);
                }
            }
        }
        // bounds: 4 columns and every RB-th row a thread
        constexpr int RB = APP_THREADS / (D / 4);
        {
            const int x = tid % (D / 4) * 4;
            int lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo[j] = 127;
                hi[j] = -127;
            }
            for (int r = tid / (D / 4); r < n; r += RB) {
                const uint32_t v = *(const uint32_t *)(kst + r * D + x);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = code_rank((v >> 8 * j) & 0xffu);
                    lo[j] = min(lo[j], k);
                    hi[j] = max(hi[j], k);
                }
            }
            if (tid / (D / 4) < n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    atomicMin(&lo_lds[x + j], lo[j]);
                    atomicMax(&hi_lds[x + j], hi[j]);
                }
        }
        __syncthreads();
        for (int x = tid; x < D; x += APP_THREADS) {
            const int lo = lo_lds[x], hi = hi_lds[x];
            const bool nan = bad_page || lo == -127;       // only a NaN bound ranks there
            auto code = [](int v) { return (uint8_t)(v < 0 ? 0x80 | -v : v); };
            bp[x] = nan ? (uint8_t)SSA_CODE_NAN : code(lo);
            bp[D + x] = nan ? (uint8_t)SSA_CODE_NAN : code(hi);
        }
        if (tid == 0) {
            c.k_scale[ph] = k_new;
            c.v_scale[ph] = v_new;
        }
    }
}

template <typename T, int D, bool VEC, int NT>
int launch_append_nt(const ssa_cache_append_args &a, int window, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(a.T, window), (unsigned)a.cache.Hkv);
    const size_t lds = (size_t)2 * a.cache.page * D;
    SSA_ALLOW_LDS((cache_append_kernel<T, D, VEC, NT>), lds);
    cache_append_kernel<T, D, VEC, NT><<<grid, NT, lds, s>>>(a, window);
    return SSA_OK;
}

template <typename T, int D>
int launch_append(const ssa_cache_append_args &a, hipStream_t s) {
    // a workgroup looks at `window` rows for the first rows of runs and serves them in
    // turn: about 1,024 workgroups in all, what the chip holds at once, whether each
    // row is a run (single tokens) or most lie inside one (prompts)
    const int64_t per = (int64_t)a.T * a.cache.Hkv / 1024;
    const int window = (int)(per < 1 ? 1 : (per > SSA_WAVE ? SSA_WAVE : per));
    // rows in 16-byte pieces (8 elements) where they all start at one
    const int64_t strides = a.k_st | a.k_sh | a.v_st | a.v_sh;
    const bool vec = a.cache.d % 8 == 0 && (strides * (int64_t)sizeof(T)) % 16 == 0 &&
                     (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
    constexpr int NT = D == 256 ? 512 : 256;   // at most 8 rows a thread
    return vec ? launch_append_nt<T, D, true, NT>(a, window, s)
               : launch_append_nt<T, D, false, NT>(a, window, s);
}

template <typename T>
int launch_append_t(const ssa_cache_append_args &a, hipStream_t s) {
    return a.cache.D == 64 ? launch_append<T, 64>(a, s)
                           : (a.cache.D == 128 ? launch_append<T, 128>(a, s)
                                               : launch_append<T, 256>(a, s));
}

// ---------------------------------------------------------------------------- select
// One workgroup per (row, kv head).  The bound of a page is one dot product of
// its two bound rows with the group's summed positive and negative parts of q, in
// fp64, so that the order is the formula's and not the summation's (products of a
// 24-bit q and a 4-bit code are exact).  D / 8 lanes read a page, four pages at a
// time: their sums fold into each other, half the lanes keeping half the pages at
// each step.  The smallest taken key is then found by its digits, from the highest
// bit in which keys differ, and the chosen pages are written in ascending order.
// Bound by latency (page ids, then bounds: 32 rows of 8 heads over up to 512 pages 14
// us) and by the conversions to fp64 (1,000 rows of 4 heads over 250 pages: 27 us).
constexpr int SEL_MAX_WIDTH = 16384;        // scores of a row in LDS

// order-preserving map of a score: NaN as +inf, an absent page 0
__device__ __forceinline__ uint64_t score_key64(double s) {
    if (s != s) s = __longlong_as_double(0x7ff0000000000000ll);
    const uint64_t u = (uint64_t)__double_as_longlong(s == 0. ? 0. : s);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(NT)
select_pages_kernel(ssa_select_pages_args a) {
    constexpr int LP = D / 8, NW = NT / SSA_WAVE;           // LP lanes of 16 codes a page
    constexpr int PARTS = NT < D ? 1 : NT / D;
    extern __shared__ uint64_t sel_keys[];
    __shared__ double qsum[PARTS * 2 * D];
    __shared__ uint32_t hist[2][256];
    __shared__ uint32_t digit, left_s, max_hi, min_hi;
    __shared__ int gt_cnt[NW], eq_cnt[NW];
    const ssa_kv_cache &c = a.cache;
    const int t = (int)blockIdx.x, h = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int lane = lane_id(), wave = tid / SSA_WAVE;
    const int rep = a.Hq / c.Hkv;
    int32_t *out = a.out + ((int64_t)t * c.Hkv + h) * a.top_k;
    const int r = a.rows.requests[t], pos = a.rows.positions[t];
    int n = 0;
    if (r >= 0 && r < a.rows.R && pos >= 0) n = min(pos / c.page + 1, a.rows.width);
    if (n <= a.top_k) {
        for (int i = tid; i < a.top_k; i += NT) out[i] = i < n ? i : -1;
        return;
    }
    // the group's sums of the negative parts of q (for the smallest key codes) and
    // of the positive ones (for the largest)
    for (int i = tid; i < PARTS * D; i += NT) {
        const int x = i % D, part = i / D;
        double p = 0., m = 0.;
        if (x < c.d)
            for (int g = part; g < rep; g += PARTS) {
                const float v =
                    to_f32(((const T *)a.q)[t * a.q_st + (int64_t)(h * rep + g) * a.q_sh + x]);
                p += (double)(v < 0.f ? 0.f : v);           // a NaN stays in both
                m += (double)(v > 0.f ? 0.f : v);
            }
        qsum[part * 2 * D + x] = m;
        qsum[part * 2 * D + D + x] = p;
    }
    for (int i = tid; i < 256; i += NT) hist[0][i] = 0;
    if (tid == 0) {
        max_hi = 0;
        min_hi = ~0u;
    }
    __syncthreads();
    if (PARTS > 1) {
        if (tid < 2 * D) {
            double v = qsum[tid];
#pragma unroll
            for (int i = 1; i < PARTS; ++i) v += qsum[i * 2 * D + tid];
            qsum[tid] = v;
        }
        __syncthreads();
    }
    const int sub = tid % LP;
    double qr[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) qr[j] = qsum[sub * 16 + j];
    const int first = min(a.first, n), last = max(n - a.recent, first);
    const int32_t *table = a.rows.block_table + (int64_t)r * a.rows.table_stride;
    uint32_t mx = 0, mn = ~0u;
    constexpr int STEP = NT / LP * 4;
    int next[4];                              // page ids, loaded an iteration ahead
#pragma unroll
    for (int i = 0; i < 4; ++i) next[i] = table[min(first + tid / LP * 4 + i, n - 1)];
    for (int p0 = first + tid / LP * 4; p0 < last; p0 += STEP) {
        int pg[4];
        uint4 w[4];
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pg[i] = p0 + i < last ? next[i] : -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t ph = (int64_t)(pg[i] >= 0 && pg[i] < c.num_pages ? pg[i] : 0) * c.Hkv + h;
            w[i] = ((const uint4 *)((const uint8_t *)c.bounds + ph * 2 * D))[sub];
            sc[i] = c.k_scale[ph];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) next[i] = table[min(p0 + STEP + i, n - 1)];
        double s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            s[i] = 0.;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)ws[j], false);
                const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)ws[j], true);
                s[i] = fma((double)lo[0], qr[4 * j], s[i]);
                s[i] = fma((double)lo[1], qr[4 * j + 1], s[i]);
                s[i] = fma((double)hi[0], qr[4 * j + 2], s[i]);
                s[i] = fma((double)hi[1], qr[4 * j + 3], s[i]);
            }
            s[i] *= (double)sc[i];
        }
        // lanes of the upper half keep pages 2 and 3, then of each quarter one page;
        // every page's sum is the same tree over its lanes
        const bool ua = sub & (LP / 2), ub = sub & (LP / 4);
        double k0 = ua ? s[2] : s[0], k1 = ua ? s[3] : s[1];
        k0 += __shfl_xor(ua ? s[0] : s[2], LP / 2, SSA_WAVE);
        k1 += __shfl_xor(ua ? s[1] : s[3], LP / 2, SSA_WAVE);
        double v = ub ? k1 : k0;
        v += __shfl_xor(ub ? k0 : k1, LP / 4, SSA_WAVE);
#pragma unroll
        for (int o = LP / 8; o > 0; o >>= 1) v += __shfl_xor(v, o, SSA_WAVE);
        const int i = (ua ? 2 : 0) + (ub ? 1 : 0), p = p0 + i;
        if (sub % (LP / 4) == 0 && p < last) {
            const int pi = i == 0 ? pg[0] : (i == 1 ? pg[1] : (i == 2 ? pg[2] : pg[3]));
            const uint64_t key = pi >= 0 && pi < c.num_pages ? score_key64(v) : 0;
            sel_keys[p - first] = key;
            mx = max(mx, (uint32_t)(key >> 32));
            mn = min(mn, (uint32_t)(key >> 32));
        }
    }
    mx = wave_max_u(mx);
    mn = wave_min_u(mn);
    if (lane == 0) {
        atomicMax(&max_hi, mx);
        atomicMin(&min_hi, mn);
    }
    __syncthreads();
    // the left-th largest of nc keys, digit by digit; the keys agree above the first
    const int nc = last - first;
    uint32_t left = (uint32_t)(a.top_k - first - (n - last));
    const uint32_t differ = max_hi ^ min_hi;
    int shift = differ ? max(32 + 31 - __clz((int)differ) - 7, 0) : 24;
    // keys >> (shift + 8) are the same for all at first
    uint64_t prefix = ((uint64_t)max_hi << 32) >> shift >> 8;
    int buf = 0, bits = 8;
    if (left > 0)
        for (;;) {
            for (int i = tid; i < nc; i += NT) {
                const uint64_t k = sel_keys[i] >> shift;
                if ((k >> bits) == prefix)
                    atomicAdd(&hist[buf][(uint32_t)k & ((1u << bits) - 1u)], 1u);
            }
            for (int i = tid; i < 256; i += NT) hist[buf ^ 1][i] = 0;
            __syncthreads();
            if (wave == 0) {                // four digits a lane, sums from the top
                uint32_t b[4], own = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) own += b[j] = hist[buf][4 * lane + j];
                uint32_t suf = own;
#pragma unroll
                for (int o = 1; o < SSA_WAVE; o <<= 1) {
                    const uint32_t u = (uint32_t)__shfl_down((int)suf, o, SSA_WAVE);
                    if (lane + o < SSA_WAVE) suf += u;
                }
                uint32_t above = suf - own;
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    if (above < left && above + b[j] >= left) {
                        digit = (uint32_t)(4 * lane + j);
                        left_s = left - above;
                    }
                    above += b[j];
                }
            }
            __syncthreads();
            left = left_s;
            prefix = (prefix << bits) | digit;
            if (shift == 0 || hist[buf][digit] == left) break;
            bits = min(shift, 8);
            shift -= bits;
            buf ^= 1;
            __syncthreads();                // digit and left are read
        }
    // taken: the forced pages, those above the prefix, the first `left` equal to it
    int gt0 = 0, eq0 = 0;
    for (int b = 0; b < n; b += NT) {
        const int p = b + tid;
        bool gt = p < n && (p < first || p >= last), eq = false;
        if (p >= first && p < last && left > 0) {
            const uint64_t k = sel_keys[p - first] >> shift;
            gt = k > prefix;
            eq = k == prefix;
        }
        const uint64_t mg = wave_ballot(gt), me = wave_ballot(eq);
        if (lane == 0) {
            gt_cnt[wave] = __popcll(mg);
            eq_cnt[wave] = __popcll(me);
        }
        __syncthreads();
        int g = gt0 + lanes_below(mg), e = eq0 + lanes_below(me);
        for (int w = 0; w < NW; ++w) {
            if (w < wave) {
                g += gt_cnt[w];
                e += eq_cnt[w];
            }
            gt0 += gt_cnt[w];
            eq0 += eq_cnt[w];
        }
        const int at = g + min(e, (int)left);
        if ((gt || (eq && e < (int)left)) && at < a.top_k) out[at] = p;
        __syncthreads();
    }
}

template <typename T, int D, int NT>
int launch_select(const ssa_select_pages_args &a, hipStream_t s) {
    const size_t lds = (size_t)a.rows.width * 8;
    SSA_ALLOW_LDS((select_pages_kernel<T, D, NT>), lds);
    const dim3 grid((unsigned)a.rows.T, (unsigned)a.cache.Hkv);
    select_pages_kernel<T, D, NT><<<grid, NT, lds, s>>>(a);
    return SSA_OK;
}

// Few rows: a CU has one workgroup or none, and 16 waves shorten its walk over the
// pages (256 of up to 500 pages: 15 us, with 4 waves 18 us; 512: 26 us and 20 us).  Many:
// a wave each, with no barriers to wait at (4,096 of 125 pages: 28 us, with 4 waves 33
// us), where the LDS holds enough of them and no wave has so many pages that the chip
// waits for the last ones (2,048 of 500: 81 us, with 4 waves 57 us; 4,096: 106 and 107).
template <typename T, int D>
int launch_select_d(const ssa_select_pages_args &a, hipStream_t s) {
    const int64_t n = (int64_t)a.rows.T * a.cache.Hkv;
    if (n <= 256) return launch_select<T, D, 1024>(a, s);
    if (n >= 2048 && a.rows.width <= (n < 8192 ? n / 8 : 1024)) return launch_select<T, D, 64>(a, s);
    return launch_select<T, D, 256>(a, s);
}

template <typename T>
int launch_select_t(const ssa_select_pages_args &a, hipStream_t s) {
    return a.cache.D == 64 ? launch_select_d<T, 64>(a, s)
                           : (a.cache.D == 128 ? launch_select_d<T, 128>(a, s)
                                               : launch_select_d<T, 256>(a, s));
}

}  // namespace

extern "C" int ssa_page_plan(const ssa_page_plan_args *a, void *stream) {
    SSA_CHECK_ARG(a, "page_plan: null arguments");
    SSA_CHECK_ARG(a->R >= 1 && a->T >= 0 && a->width >= 1 && a->table_stride >= a->width,
                  "page_plan: R=%d T=%d width=%d table_stride=%lld", a->R, a->T, a->width,
                  (long long)a->table_stride);
    if (a->R > PLAN_MAX_R) {
        ssa_set_error("page_plan: %d requests (at most %d)", a->R, PLAN_MAX_R);
        return SSA_E_UNSUP;
    }
    if (a->page != 32 && a->page != 64 && a->page != 128) {
        ssa_set_error("page_plan: pages of %d tokens (32, 64 or 128)", a->page);
        return SSA_E_UNSUP;
    }
    SSA_CHECK_ARG((int64_t)a->width * a->page < (1ll << 31),
                  "page_plan: %d pages of %d tokens pass 2^31 positions", a->width, a->page);
    SSA_CHECK_ARG(a->free_capacity >= 0 && (a->free_capacity == 0 || a->free_pages),
                  "page_plan: free list");
    SSA_CHECK_ARG(a->cached && a->new_rows && a->block_table && a->free_count && a->starts &&
                      a->lengths && a->free_count_out && a->refused &&
                      (a->T == 0 || (a->slots && a->positions && a->requests)),
                  "page_plan: null pointer");
    const hipStream_t s = (hipStream_t)stream;
    const int rc = a->R <= PLAN_THREADS       ? launch_plan<1>(*a, s)
                   : a->R <= 4 * PLAN_THREADS ? launch_plan<4>(*a, s)
                   : a->R <= 16 * PLAN_THREADS ? launch_plan<16>(*a, s)
                                               : launch_plan<64>(*a, s);
    if (rc != SSA_OK) return rc;
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}

extern "C" int ssa_cache_append(const ssa_cache_append_args *a, void *stream) {
    SSA_CHECK_ARG(a, "cache_append: null arguments");
    const int rc = ssa_check_cache(&a->cache);
    if (rc != SSA_OK) return rc;
    SSA_CHECK_ARG(a->dtype == SSA_F32 || a->dtype == SSA_BF16 || a->dtype == SSA_F16,
                  "cache_append: dtype %d", a->dtype);
    SSA_CHECK_ARG(a->T >= 0, "cache_append: T=%d", a->T);
    if (a->T == 0) return SSA_OK;
    SSA_CHECK_ARG(a->k && a->v && a->slots, "cache_append: null pointer");
    const hipStream_t s = (hipStream_t)stream;
    const int lc = a->dtype == SSA_F32 ? launch_append_t<float>(*a, s)
                 : a->dtype == SSA_BF16 ? launch_append_t<bf16_t>(*a, s)
                                        : launch_append_t<f16_t>(*a, s);
    if (lc != SSA_OK) return lc;
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}

extern "C" int ssa_select_pages(const ssa_select_pages_args *a, void *stream) {
    SSA_CHECK_ARG(a, "select_pages: null arguments");
    int rc = ssa_check_cache(&a->cache);
    if (rc != SSA_OK) return rc;
    rc = ssa_check_rows(&a->rows, &a->cache);
    if (rc != SSA_OK) return rc;
    SSA_CHECK_ARG(a->dtype == SSA_F32 || a->dtype == SSA_BF16 || a->dtype == SSA_F16,
                  "select_pages: dtype %d", a->dtype);
    SSA_CHECK_ARG(a->Hq >= 1 && a->Hq % a->cache.Hkv == 0,
                  "select_pages: %d query heads are not a multiple of %d kv heads", a->Hq,
                  a->cache.Hkv);
    SSA_CHECK_ARG(a->first >= 0 && a->recent >= 1 && (int64_t)a->first + a->recent <= a->top_k,
                  "select_pages: first=%d recent=%d top_k=%d (recent >= 1, both within top_k)",
                  a->first, a->recent, a->top_k);
    if (a->rows.width > SEL_MAX_WIDTH) {
        ssa_set_error("select_pages: tables of %d pages (at most %d)", a->rows.width,
                      SEL_MAX_WIDTH);
        return SSA_E_UNSUP;
    }
    if (a->rows.T == 0) return SSA_OK;
    SSA_CHECK_ARG(a->q && a->out, "select_pages: null pointer");
    const hipStream_t s = (hipStream_t)stream;
    rc = a->dtype == SSA_F32 ? launch_select_t<float>(*a, s)
       : a->dtype == SSA_BF16 ? launch_select_t<bf16_t>(*a, s)
                              : launch_select_t<f16_t>(*a, s);
    if (rc != SSA_OK) return rc;
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}
