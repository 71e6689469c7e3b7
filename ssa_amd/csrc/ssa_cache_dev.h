// ssa_cache_dev.h -- what the kernels of the paged 8-bit cache share.
#pragma once

#include "ssa_common.h"

// Scales are powers of two 2^-100 .. 2^112; a magnitude of 2^120 or more counts
// as not finite (its code times a scale would leave fp32's range).
#define SSA_CACHE_E_MIN (-100)
#define SSA_CACHE_E_MAX 112
#define SSA_CACHE_TOO_BIG 1.329227995784916e36f     // 2^120

#define SSA_CODE_NAN 0x7Fu

// a cached number: e4m3 code in byte SEL of a word
template <int SEL>
__device__ __forceinline__ float code_f32(uint32_t w) {
    return __builtin_amdgcn_cvt_f32_fp8((int)w, SEL);
}

// two numbers of magnitude <= 448 as codes in bits 0..15, to nearest, ties to even
__device__ __forceinline__ uint32_t codes2(float a, float b) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// a word's codes times a power of two <= 1, rounded again
__device__ __forceinline__ uint32_t codes4_scaled(uint32_t w, float f) {
    return codes4(code_f32<0>(w) * f, code_f32<1>(w) * f, code_f32<2>(w) * f, code_f32<3>(w) * f);
}

inline int ssa_cache_store_dim(int d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }

// what every entry point asks of a cache
inline int ssa_check_cache(const ssa_kv_cache *c) {
    SSA_CHECK_ARG(c->k_codes && c->v_codes && c->bounds && c->k_scale && c->v_scale,
                  "cache: null buffer");
    SSA_CHECK_ARG(c->num_pages >= 1 && c->Hkv >= 1 && c->Hkv <= 65535,
                  "cache: num_pages=%lld Hkv=%d (at least 1; at most 65535 heads)",
                  (long long)c->num_pages, c->Hkv);
    SSA_CHECK_ARG(c->num_pages <= (1ll << 31) - 1, "cache: num_pages=%lld beyond 2^31 - 1",
                  (long long)c->num_pages);
    if (c->page != 32 && c->page != 64 && c->page != 128) {
        ssa_set_error("cache: pages of %d tokens (32, 64 or 128)", c->page);
        return SSA_E_UNSUP;
    }
    if (c->d < 1 || c->d > 256 || c->D != ssa_cache_store_dim(c->d)) {
        ssa_set_error("cache: head dim %d stored as %d (1..256, stored as 64, 128 or 256)", c->d,
                      c->D);
        return SSA_E_UNSUP;
    }
    SSA_CHECK_ARG((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->bounds) & 15) == 0,
                  "cache: codes and bounds must be 16-byte aligned");
    return SSA_OK;
}

inline int ssa_check_rows(const ssa_batch_rows *r, const ssa_kv_cache *c) {
    SSA_CHECK_ARG(r->T >= 0 && r->R >= 1 && r->width >= 1 && r->table_stride >= r->width,
                  "rows: T=%d R=%d width=%d table_stride=%lld", r->T, r->R, r->width,
                  (long long)r->table_stride);
    SSA_CHECK_ARG((int64_t)r->width * c->page < (1ll << 31),
                  "rows: %d pages of %d tokens pass 2^31 positions", r->width, c->page);
    SSA_CHECK_ARG(r->block_table && r->starts && (r->T == 0 || (r->requests && r->positions)),
                  "rows: null pointer");
    return SSA_OK;
}
