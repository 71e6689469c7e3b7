// ssa_cache_attend_dev.h -- what the attention kernels over the paged cache share.
#pragma once

#include "ssa_cache_dev.h"

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;

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
            int hi = p.R;                     // last r whose first unit is <= u
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((int64_t)p.starts[mid] * p.rep / CT + mid <= u) lo = mid;
                else hi = mid - 1;
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

// launches of ssa_cache_prompt.hip: requests with more columns than `many`
int ssa_cache_prompt_columns(int dtype, int D);         // of a workgroup
void ssa_cache_prompt_launch(const AttendParams &p, int dtype, int D, int KT, hipStream_t st);
