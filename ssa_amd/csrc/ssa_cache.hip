// ssa_cache.hip -- block tables, the append and the page selection of the paged
// 8-bit key/value cache (the attention over it is in ssa_cache_attend.hip).
#include "ssa_cache_dev.h"

namespace {

// ---------------------------------------------------------------------------- plan
// Everything follows from two prefix sums over the requests (their rows, and the
// pages they need), so every workgroup forms both in its LDS and then serves its
// share of the rows by binary search: one launch, no pass between workgroups.
// Bound by latency: two block scans and log2(R) LDS reads per row.
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

__global__ void __launch_bounds__(PLAN_THREADS)
page_plan_kernel(ssa_page_plan_args a) {
    extern __shared__ uint32_t plan_lds[];
    __shared__ uint32_t part[PLAN_THREADS / SSA_WAVE];
    __shared__ uint32_t n_taken, n_refused;
    uint32_t *end = plan_lds;               // rows up to and with request r
    int32_t *base = (int32_t *)plan_lds + a.R;   // pages taken before r, -1 where refused
    const int per = (a.R + PLAN_THREADS - 1) / PLAN_THREADS;
    const int r0 = min((int)threadIdx.x * per, a.R), r1 = min(r0 + per, a.R);
    const bool first_wg = blockIdx.x == 0;
    if (threadIdx.x == 0) n_taken = n_refused = 0;
    uint32_t sum = 0, total;
    for (int r = r0; r < r1; ++r) sum = sat_add(sum, (uint32_t)max(a.new_rows[r], 0));
    uint32_t run = block_scan(sum, part, &total);
    uint32_t need = 0;
    for (int r = r0; r < r1; ++r) {
        const int c = a.cached[r], n = a.new_rows[r];
        if (first_wg) a.starts[r] = (int32_t)run;
        run = sat_add(run, (uint32_t)max(n, 0));
        end[r] = run;
        const int64_t want = ((int64_t)c + n + a.page - 1) / a.page;
        const bool fits = c >= 0 && n >= 0 && want <= a.width && run <= (uint32_t)a.T;
        const int nd = fits ? (int)(want - ((int64_t)c + a.page - 1) / a.page) : -1;
        base[r] = nd;
        need = sat_add(need, (uint32_t)max(nd, 0));
    }
    if (first_wg && threadIdx.x == 0) a.starts[a.R] = (int32_t)total;
    uint32_t upto = block_scan(need, part, &total);
    const uint32_t nfree = (uint32_t)max(0, min(*a.free_count, a.free_capacity));
    uint32_t taken = 0, refused = 0;
    for (int r = r0; r < r1; ++r) {
        const int nd = base[r];
        const uint32_t before = upto;
        upto = sat_add(upto, (uint32_t)max(nd, 0));
        const bool ok = nd == 0 || (nd > 0 && upto <= nfree);
        base[r] = ok ? (int32_t)min(before, nfree) : -1;
        taken += ok ? (uint32_t)nd : 0u;
        refused += ok ? 0u : 1u;
        if (first_wg) a.lengths[r] = a.cached[r] + (ok ? a.new_rows[r] : 0);
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
            const int c = a.cached[lo];
            req = lo;
            pos = c + (int32_t)(t - (lo ? end[lo - 1] : 0));
            const int col = pos / a.page, off = pos - col * a.page;
            const int had = (c + a.page - 1) / a.page;
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

// ---------------------------------------------------------------------------- append
// One workgroup per run of adjacent rows of one page and kv head: the run's
// largest magnitudes first (the page's scale has to hold before any code is
// rounded), then the codes, staged in LDS so that the transposed value codes go
// out in words of four tokens.  Reads every row twice, the second time from the
// L2.  Bound by latency for single tokens, by HBM for prompts.
constexpr int APP_THREADS = 256;

template <typename T>
__device__ __forceinline__ float row_elem(const void *p, int64_t i) {
    return to_f32(((const T *)p)[i]);
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

template <typename T>
__global__ void __launch_bounds__(APP_THREADS)
cache_append_kernel(ssa_cache_append_args a, int window) {
    extern __shared__ uint4 app_lds[];
    __shared__ uint32_t kmax[128], vmax[128];     // bits of each row's largest magnitude
    __shared__ uint32_t page_max[2], any_bad;
    const ssa_kv_cache &c = a.cache;
    const int h = (int)blockIdx.y, ps = c.page, D = c.D, d = c.d, tid = (int)threadIdx.x;
    const int64_t cap = c.num_pages * ps;
    uint8_t *kst = (uint8_t *)app_lds, *vst = kst + ps * D;      // [row][D] codes
    for (int w = 0; w < window; ++w) {
        const int64_t t0 = (int64_t)blockIdx.x * window + w;
        if (t0 >= a.T) break;
        const int64_t slot = a.slots[t0];
        if (slot < 0 || slot >= cap) continue;
        const int64_t pg = slot / ps;
        const int off = (int)(slot - pg * ps);
        if (off != 0 && t0 > 0 && a.slots[t0 - 1] == slot - 1) continue;   // inside a run
        // length of the run: rows t0 + i at slot + i within the page
        const int most = (int)min((int64_t)(ps - off), a.T - t0);
        int n = 1;
        for (int b = 0; b < most; b += SSA_WAVE) {
            const int i = b + lane_id();
            const uint64_t m = wave_ballot(i < most && a.slots[t0 + i] == slot + i);
            n = b + (m == ~0ull ? SSA_WAVE : __ffsll((unsigned long long)~m) - 1);
            if (m != ~0ull) break;
        }
        n = min(n, most);
        __syncthreads();                                   // the last run's LDS is read
        if (tid < 128) kmax[tid] = vmax[tid] = 0;
        if (tid < 2) page_max[tid] = 0;
        if (tid == 2) any_bad = 0;
        __syncthreads();
        const int64_t krow = t0 * a.k_st + (int64_t)h * a.k_sh;
        const int64_t vrow = t0 * a.v_st + (int64_t)h * a.v_sh;
        for (int i = tid; i < n * d; i += APP_THREADS) {
            const int r = i / d, x = i - r * d;
            // a NaN's bits, its sign cleared, are larger than every number's
            atomicMax(&kmax[r], __float_as_uint(row_elem<T>(a.k, krow + r * a.k_st + x)) & 0x7fffffffu);
            atomicMax(&vmax[r], __float_as_uint(row_elem<T>(a.v, vrow + r * a.v_st + x)) & 0x7fffffffu);
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
        const int64_t ph = pg * c.Hkv + h;
        const float k_old = off ? c.k_scale[ph] : 0.f, v_old = off ? c.v_scale[ph] : 0.f;
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
            const int words = (off + 3) / 4;               // of each channel's tokens
            for (int i = tid; i < D * words; i += APP_THREADS) {
                const int x = i / words, q = i - x * words;
                uint32_t *at = p + x * (ps / 4) + q;
                const uint32_t was = *at, now = codes4_scaled(was, f);
                const int keep = min(off - 4 * q, 4) * 8;  // bits of tokens below the run
                const uint32_t m = keep == 32 ? ~0u : (1u << keep) - 1u;
                *at = (now & m) | (was & ~m);
            }
        }
        const float ki = 1.f / k_new, vi = 1.f / v_new;    // exact
        for (int i = tid; i < n * (D / 2); i += APP_THREADS) {
            const int r = i / (D / 2), x = 2 * (i - r * (D / 2));
            const bool bad = kmax[r] == 0xffffffffu;
            const int64_t ko = krow + r * a.k_st + x, vo = vrow + r * a.v_st + x;
            const float k0 = x < d ? row_elem<T>(a.k, ko) : 0.f;
            const float k1 = x + 1 < d ? row_elem<T>(a.k, ko + 1) : 0.f;
            const float v0 = x < d ? row_elem<T>(a.v, vo) : 0.f;
            const float v1 = x + 1 < d ? row_elem<T>(a.v, vo + 1) : 0.f;
            *(uint16_t *)(kst + r * D + x) =
                (uint16_t)(bad ? SSA_CODE_NAN * 0x101u : codes2(k0 * ki, k1 * ki));
            *(uint16_t *)(vst + r * D + x) = (uint16_t)(bad ? 0u : codes2(v0 * vi, v1 * vi));
        }
        __syncthreads();
        for (int i = tid; i < n * D / 16; i += APP_THREADS)
            ((uint4 *)(kp + (int64_t)off * D))[i] = ((const uint4 *)kst)[i];
        const int q0 = off / 4, q1 = (off + n + 3) / 4;    // words of a channel's tokens
        for (int i = tid; i < D * (q1 - q0); i += APP_THREADS) {
            const int x = i % D, q = q0 + i / D;
            uint32_t v = 0;
            bool whole = true;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 4 * q + j - off;
                if (r >= 0 && r < n) v |= (uint32_t)vst[r * D + x] << (8 * j);
                else whole = false;
            }
            uint8_t *at = vp + (int64_t)x * ps + 4 * q;
            if (whole) {
                *(uint32_t *)at = v;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 4 * q + j - off;
                    if (r >= 0 && r < n) at[j] = (uint8_t)(v >> (8 * j));
                }
            }
        }
        // bounds: a code's order is that of its sign and magnitude
        for (int x = tid; x < D; x += APP_THREADS) {
            int lo = 127, hi = -127;
            bool nan = any_bad != 0;
            auto note = [&](uint32_t code) {
                const int v = (code & 0x80u) ? -(int)(code & 0x7fu) : (int)code;
                nan |= (code & 0x7fu) == SSA_CODE_NAN;
                lo = min(lo, v);
                hi = max(hi, v);
            };
            if (off) {
                const float f = k_old / k_new;
                note(codes2(code_f32<0>(bp[x]) * f, 0.f) & 0xffu);
                note(codes2(code_f32<0>(bp[D + x]) * f, 0.f) & 0xffu);
            }
            for (int r = 0; r < n; ++r) note(kst[r * D + x]);
            auto code = [&](int v) {
                return (uint8_t)(nan ? SSA_CODE_NAN : (v < 0 ? 0x80u | (uint32_t)-v : (uint32_t)v));
            };
            bp[x] = code(lo);
            bp[D + x] = code(hi);
        }
        if (tid == 0) {
            c.k_scale[ph] = k_new;
            c.v_scale[ph] = v_new;
        }
    }
}

// ---------------------------------------------------------------------------- select
// One workgroup per (row, kv head).  The bound of a page is one dot product of
// its two bound rows with the group's summed positive and negative parts of q;
// fp64, so that the order is the formula's and not the summation's (products of a
// 24-bit q and a 4-bit code are exact).  The top_k-th score is then found by its
// bits, and the chosen pages written in ascending order.
constexpr int SEL_THREADS = 256;
constexpr int SEL_MAX_WIDTH = 16384;        // scores of a row in LDS

// order-preserving map of a score: NaN as +inf, an absent page 0
__device__ __forceinline__ uint64_t score_key64(double s) {
    if (s != s) s = __longlong_as_double(0x7ff0000000000000ll);
    const uint64_t u = (uint64_t)__double_as_longlong(s == 0. ? 0. : s);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

template <typename T, int D>
__global__ void __launch_bounds__(SEL_THREADS)
select_pages_kernel(ssa_select_pages_args a) {
    extern __shared__ uint64_t sel_keys[];
    __shared__ double qsum[2 * D];
    __shared__ uint32_t hist[256];
    __shared__ uint32_t digit, left_s;
    __shared__ int wave_cnt[SEL_THREADS / SSA_WAVE];
    const ssa_kv_cache &c = a.cache;
    const int t = (int)blockIdx.x, h = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int rep = a.Hq / c.Hkv;
    int32_t *out = a.out + ((int64_t)t * c.Hkv + h) * a.top_k;
    const int r = a.rows.requests[t], pos = a.rows.positions[t];
    int n = 0;
    if (r >= 0 && r < a.rows.R && pos >= 0) n = min(pos / c.page + 1, a.rows.width);
    if (n <= a.top_k) {
        for (int i = tid; i < a.top_k; i += SEL_THREADS) out[i] = i < n ? i : -1;
        return;
    }
    // group's sums of the positive parts (for hi) and the negative ones (for lo)
    for (int x = tid; x < D; x += SEL_THREADS) {
        double p = 0., m = 0.;
        if (x < c.d)
            for (int g = 0; g < rep; ++g) {
                const float v = to_f32(((const T *)a.q)[t * a.q_st + (int64_t)(h * rep + g) * a.q_sh + x]);
                if (v != v) p = m = (double)v;              // NaN stays
                else if (v > 0.f) p += (double)v;
                else m += (double)v;
            }
        qsum[x] = m;
        qsum[D + x] = p;
    }
    __syncthreads();
    const int first = min(a.first, n), last = max(n - a.recent, first);
    constexpr int LP = D / 8;                               // lanes of a page: 16 codes each
    const int sub = tid % LP;
    double qr[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) qr[j] = qsum[sub * 16 + j];
    const int32_t *table = a.rows.block_table + (int64_t)r * a.rows.table_stride;
    for (int p = first + tid / LP; p < last; p += SEL_THREADS / LP) {
        const int pg = table[p];
        const bool there = pg >= 0 && pg < c.num_pages;
        double s = 0.;
        if (there) {
            const int64_t ph = (int64_t)pg * c.Hkv + h;
            const uint4 w = ((const uint4 *)((const uint8_t *)c.bounds + ph * 2 * D))[sub];
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s = fma((double)code_f32<0>(ws[j]), qr[4 * j], s);
                s = fma((double)code_f32<1>(ws[j]), qr[4 * j + 1], s);
                s = fma((double)code_f32<2>(ws[j]), qr[4 * j + 2], s);
                s = fma((double)code_f32<3>(ws[j]), qr[4 * j + 3], s);
            }
            s *= (double)c.k_scale[ph];
        }
#pragma unroll
        for (int o = LP / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, SSA_WAVE);
        if (sub == 0) sel_keys[p - first] = there ? score_key64(s) : 0;
    }
    __syncthreads();
    // the need-th largest key among nc, and how many equal to it are taken
    const int nc = last - first;
    uint32_t left = (uint32_t)(a.top_k - first - (n - last));
    uint64_t prefix = 0;
    int shift = 56;
    if (left > 0)
    for (;; shift -= 8) {
        hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < nc; i += SEL_THREADS) {
            const uint64_t k = sel_keys[i];
            if (shift == 56 || (k >> (shift + 8)) == prefix)
                atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        // digit: the largest v with sum of hist[v..] >= left
        uint32_t above = 0;
        for (int v = tid + 1; v < 256; ++v) above += hist[v];
        if (above < left && above + hist[tid] >= left) {
            digit = (uint32_t)tid;
            left_s = left - above;
        }
        __syncthreads();
        left = left_s;
        prefix = (prefix << 8) | digit;
        const bool done = shift == 0 || hist[digit] == left;
        __syncthreads();
        if (done) break;
    }
    // pages above the prefix are taken, and the first `left` equal to it
    int out_n = 0;
    uint32_t eq_n = 0;
    for (int b = 0; b < n; b += SEL_THREADS) {
        const int p = b + tid;
        bool take = p < n && (p < first || p >= last), eq = false;
        if (p >= first && p < last && left > 0) {
            const uint64_t k = sel_keys[p - first] >> shift;
            take = k > prefix;
            eq = k == prefix;
        }
        // ranks by two scans: of the equal ones, then of those taken
        const int wave = tid / SSA_WAVE;
        uint64_t m = wave_ballot(eq);
        if (lane_id() == 0) wave_cnt[wave] = __popcll(m);
        __syncthreads();
        uint32_t er = eq_n + (uint32_t)lanes_below(m), ea = 0;
        for (int w = 0; w < SEL_THREADS / SSA_WAVE; ++w) {
            if (w < wave) er += (uint32_t)wave_cnt[w];
            ea += (uint32_t)wave_cnt[w];
        }
        eq_n += ea;
        take = take || (eq && er < left);
        __syncthreads();
        m = wave_ballot(take);
        if (lane_id() == 0) wave_cnt[wave] = __popcll(m);
        __syncthreads();
        int at = out_n + lanes_below(m), all = 0;
        for (int w = 0; w < SEL_THREADS / SSA_WAVE; ++w) {
            if (w < wave) at += wave_cnt[w];
            all += wave_cnt[w];
        }
        out_n += all;
        if (take && at < a.top_k) out[at] = p;
        __syncthreads();
    }
    for (int i = out_n + tid; i < a.top_k; i += SEL_THREADS) out[i] = -1;
}

template <typename T>
void launch_select(const ssa_select_pages_args &a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows.T, (unsigned)a.cache.Hkv);
    const size_t lds = (size_t)a.rows.width * 8;
    if (a.cache.D == 64) select_pages_kernel<T, 64><<<grid, SEL_THREADS, lds, s>>>(a);
    else if (a.cache.D == 128) select_pages_kernel<T, 128><<<grid, SEL_THREADS, lds, s>>>(a);
    else select_pages_kernel<T, 256><<<grid, SEL_THREADS, lds, s>>>(a);
}

template <typename T>
int allow_select_lds(size_t lds) {
    SSA_ALLOW_LDS((select_pages_kernel<T, 64>), lds);
    SSA_ALLOW_LDS((select_pages_kernel<T, 128>), lds);
    SSA_ALLOW_LDS((select_pages_kernel<T, 256>), lds);
    return SSA_OK;
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
    const size_t lds = (size_t)a->R * 8;
    SSA_ALLOW_LDS(page_plan_kernel, lds);
    // workgroups enough for four rows a thread, at most two per CU
    const int64_t want = ceil_div(a->T, PLAN_THREADS * 4);
    const int grid = (int)(want < 1 ? 1 : (want > 512 ? 512 : want));
    page_plan_kernel<<<grid, PLAN_THREADS, lds, (hipStream_t)stream>>>(*a);
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
    // a workgroup looks at `window` rows for the first rows of runs: one each while
    // they all may be (single tokens), more where most lie inside a run
    const int window = a->T <= 1024 ? 1 : (a->T <= 4096 ? 4 : 16);
    const dim3 grid((unsigned)ceil_div(a->T, window), (unsigned)a->cache.Hkv);
    const size_t lds = (size_t)2 * a->cache.page * a->cache.D;
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == SSA_F32) {
        SSA_ALLOW_LDS(cache_append_kernel<float>, lds);
        cache_append_kernel<float><<<grid, APP_THREADS, lds, s>>>(*a, window);
    } else if (a->dtype == SSA_BF16) {
        SSA_ALLOW_LDS(cache_append_kernel<bf16_t>, lds);
        cache_append_kernel<bf16_t><<<grid, APP_THREADS, lds, s>>>(*a, window);
    } else {
        SSA_ALLOW_LDS(cache_append_kernel<f16_t>, lds);
        cache_append_kernel<f16_t><<<grid, APP_THREADS, lds, s>>>(*a, window);
    }
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
    const size_t lds = (size_t)a->rows.width * 8;
    const hipStream_t s = (hipStream_t)stream;
    if (a->dtype == SSA_F32) {
        rc = allow_select_lds<float>(lds);
        if (rc != SSA_OK) return rc;
        launch_select<float>(*a, s);
    } else if (a->dtype == SSA_BF16) {
        rc = allow_select_lds<bf16_t>(lds);
        if (rc != SSA_OK) return rc;
        launch_select<bf16_t>(*a, s);
    } else {
        rc = allow_select_lds<f16_t>(lds);
        if (rc != SSA_OK) return rc;
        launch_select<f16_t>(*a, s);
    }
    SSA_CHECK_LAUNCH();
    return SSA_OK;
}
