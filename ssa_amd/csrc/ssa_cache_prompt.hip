// ssa_cache_prompt.hip -- attention over the paged 8-bit cache for many query rows
// of one request (prompts and their chunks).
//
// The products and the mapping of keys to lanes are those of ssa_cache_attend.hip
// (S^T = K Q^T, O^T = V^T P^T, a column is a query row, P^T stays in registers).
// Here each wave owns 16 columns and walks every key tile of the workgroup's
// range, so the tiles are shared: the waves convert a tile's codes to 16-bit floats
// once, into LDS, in the order in which the matrix operands read them (a fragment is
// 64 slots of 16 bytes: every LDS access is free of conflicts), double-buffered, with
// the codes of the two tiles behind on their way from memory.  Bound by instruction
// issue: of a 4,096-token prompt's time (32 / 8 heads, d 128, bf16: 172 us, 797 TFLOP/s)
// the vector unit is busy 41%, the matrix unit 33%.
#include "ssa_cache_attend_dev.h"

namespace {

// 16-byte pieces of LDS a workgroup uses
template <int D, int KT> constexpr int prompt_lds() {
    return 2 * 2 * (KT / 16 * (D / 64) + D / 16 * (KT / 32) / 2) * SSA_WAVE + 2;
}

// Waves of a workgroup, 16 columns each: four a SIMD where the registers allow it
// (two workgroups a CU), which hides what one wave's softmax waits for better than
// wider waves did (4 waves of 32 columns: 186 us for a prompt of 4,096 tokens).
template <typename T, int D> constexpr int prompt_waves() { return sizeof(T) == 4 && D == 256 ? 4 : 8; }

template <typename T, int D, int KT>
__device__ __forceinline__ void prompt_unit(const AttendParams &p, unsigned block, int split, u32x4 *lds) {
    constexpr int PW = prompt_waves<T, D>();
    typedef Columns<T, D, KT> C;
    typedef typename C::QV QV;
    typedef typename C::PV PV;
    constexpr int NQ = C::NQ, NP = C::NP, NB = C::NB, DP = C::DP, ND = C::ND, KS = C::KS;
    constexpr int CT = PW * 16;
    // a load unit: 16 codes a lane, two fragments
    constexpr int KU = NB * DP, VU = ND * KS / 2, NU = KU + VU, UW = NU < PW ? 1 : NU / PW;
    u32x4 (*frag)[2 * NU][SSA_WAVE] = (u32x4 (*)[2 * NU][SSA_WAVE])lds;    // two buffers
    int *most_lds = (int *)(lds + prompt_lds<D, KT>() - 2);

    const int lane = lane_id(), lrow = lane >> 2, lpiece = lane & 3;
    const int to = slot_of(lrow, lpiece), from = slot_of(lane & 15, lane >> 4);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    // kv heads run fastest: an XCD's workgroups share their heads' pages in its L2;
    // units run backwards, those with the most keys first
    const int h = (int)(block % (unsigned)p.Hkv);
    const int u = p.units - 1 - (int)(block / (unsigned)p.Hkv);
    Unit un;
    if (!locate_unit(p, u, CT, un)) return;
    const int wc0 = un.c0 + wave * 16;        // this wave's first column
    C w;
    w.start(p, un, wc0, un.c1, h);
    if (lane == 0) most_lds[wave] = w.most;
    __syncthreads();
    int most_wg = -1;
#pragma unroll
    for (int i = 0; i < PW; ++i) most_wg = max(most_wg, most_lds[i]);
    most_wg = __builtin_amdgcn_readfirstlane(most_wg);

    const int page = 1 << p.page_shift;
    const int n_tiles = most_wg < 0 ? 0 : most_wg / KT + 1;
    const int tile0 = split * p.chunk, tile1 = min(tile0 + p.chunk, n_tiles);
    const int sub_shift = p.page_shift - (KT == 64 ? 6 : 5);
    const int32_t *table = p.table + (int64_t)(un.req < 0 ? 0 : un.req) * p.table_stride;

    // this wave's load units: 64 columns of a key block, or 16 value rows (two times 16
    // of half the tokens); the first half of the waves take keys, the others values
    const int u0 = wave * UW;
    const bool stages = u0 < NU, keys = u0 < KU;
    int off[UW];
    u32x4 raw[2][UW];                         // of the next two tiles
#pragma unroll
    for (int x = 0; x < UW; ++x) {
        const int b = (u0 + x) / DP, i = (u0 + x) % DP, v = u0 + x - KU;
        off[x] = keys ? (KT / 4 * (lrow >> 2) + 4 * b + (lrow & 3)) * D + i * 64 + lpiece * 16
                      : KT == 64 ? ((v * 16 + lrow) << p.page_shift) + 16 * lpiece
                                 : ((v * 32 + lrow) << p.page_shift) + 8 * lpiece;
    }
    struct Tile { int pg; float ks, vs; };
    // A tile's table entry is loaded a tile ahead of its codes, whatever it is (of the
    // last tile, past the end), and judged where they are: nothing waits for it.
    const int last_entry = (max(tile1, 1) - 1) >> sub_shift;
    auto entry = [&](int tile) { return table[min(tile >> sub_shift, last_entry)]; };
    auto fetch = [&](u32x4 (&raw)[UW], int tile, int pg, Tile &ti) {
        ti.pg = tile < tile1 && pg >= 0 && pg < p.num_pages ? pg : -1;
        if (ti.pg < 0) return;
        const int sub = tile & ((1 << sub_shift) - 1);
        const int64_t ph = (int64_t)pg * p.Hkv + h;
        ti.ks = p.ks[ph];
        ti.vs = p.vs[ph];
        if (!stages) return;
        const uint8_t *at = keys ? p.k + ph * D * page + sub * KT * D : p.v + ph * D * page + sub * KT;
        if (KT == 64 || keys) {
#pragma unroll
            for (int x = 0; x < UW; ++x) raw[x] = *(const u32x4 *)(at + off[x]);
        } else {
#pragma unroll
            for (int x = 0; x < UW; ++x) {
                const u32x2 a = *(const u32x2 *)(at + off[x]);
                const u32x2 b = *(const u32x2 *)(at + off[x] + (16 << p.page_shift));
                raw[x] = u32x4{a.x, a.y, b.x, b.y};
            }
        }
    };
    auto stage = [&](int buf, const u32x4 (&raw)[UW], const Tile &ti) {
        if (ti.pg < 0 || !stages) return;
        u32x4 *f = &frag[buf][2 * u0][to];
        if (keys) {
#pragma unroll
            for (int x = 0; x < UW; ++x) {
                *(QV *)(f + 2 * x * SSA_WAVE) = Ops<T>::key(raw[x].x, raw[x].y);
                *(QV *)(f + (2 * x + 1) * SSA_WAVE) = Ops<T>::key(raw[x].z, raw[x].w);
            }
        } else {
#pragma unroll
            for (int x = 0; x < UW; ++x) {
                *(PV *)(f + 2 * x * SSA_WAVE) = Ops<T>::value(raw[x].x, raw[x].y, ti.vs);
                *(PV *)(f + (2 * x + 1) * SSA_WAVE) = Ops<T>::value(raw[x].z, raw[x].w, ti.vs);
            }
        }
    };

    Tile cur{-1, 0.f, 0.f}, nxt{-1, 0.f, 0.f}, far{-1, 0.f, 0.f};
    int entry3 = -1;
    if (tile0 < tile1) {
        const int pg0 = entry(tile0), pg1 = entry(tile0 + 1), pg2 = entry(tile0 + 2);
        entry3 = entry(tile0 + 3);
        fetch(raw[1], tile0, pg0, cur);
        fetch(raw[0], tile0 + 1, pg1, nxt);
        stage(0, raw[1], cur);
        fetch(raw[1], tile0 + 2, pg2, far);
    }
    __syncthreads();
    for (int tile2 = tile0; tile2 < tile1; tile2 += 2)
#pragma unroll
    for (int buf = 0; buf < 2; ++buf) {       // LDS buffer of the tile, registers of the next
        const int tile = tile2 + buf;
        if (tile >= tile1) break;
        stage(buf ^ 1, raw[buf], nxt);
        Tile nn{-1, 0.f, 0.f};
        fetch(raw[buf], tile + 3, entry3, nn);
        entry3 = entry(tile + 4);
        const int key0 = tile * KT;
        if (cur.pg >= 0 && key0 <= w.most) {
            f32x4 s[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
            const u32x4 *kl = &frag[buf][0][from], *vl = &frag[buf][2 * KU][from];
#pragma unroll
            for (int k = 0; k < DP * 2; ++k)   // neighbouring products are independent
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const QV kf = *(const QV *)(kl + (b * DP * 2 + k) * SSA_WAVE);
#pragma unroll
                    for (int n = NQ - 1; n >= 0; --n) s[b] = mfma(kf, w.q[k][n], s[b]);
                }
            PV pf[KS][NP];
            if (w.softmax(s, cur.ks, cur.vs, key0, pf))
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const PV vf = *(const PV *)(vl + (i * KS + k) * SSA_WAVE);
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n) w.o[i] = mfma(vf, pf[k][n], w.o[i]);
                    }
        }
        __syncthreads();
        cur = nxt;
        nxt = far;
        far = nn;
    }
    w.finish(p, un, wc0, un.c1, h, split, tile0 < tile1);
}

// Requests with few columns (p, first) and with many (q) in one launch, each kind in
// its own number of chunks; the lengths, and so which there are, are known on the GPU
// alone.
template <typename T, int D, int KT>
__global__ void __launch_bounds__((prompt_waves<T, D>() * SSA_WAVE),
                                  (sizeof(T) == 4 && D == 256 ? 1 : (sizeof(T) == 2 && D <= 128 ? 4 : 2)))
cache_prompt_kernel(AttendParams p, int many_units, int many_S, int many_chunk, float *many_ml,
                    float *many_o) {
    __shared__ u32x4 lds[prompt_lds<D, KT>()];
    unsigned b = blockIdx.x;
    const unsigned few = (unsigned)(p.units * p.Hkv) * (unsigned)p.S;
    if (b >= few) {
        b -= few;
        p.mode = UNITS_MANY;
        p.units = many_units;
        p.S = many_S;
        p.chunk = many_chunk;
        p.part_ml = many_ml;
        p.part_o = many_o;
    }
    const unsigned per = (unsigned)(p.units * p.Hkv);
    prompt_unit<T, D, KT>(p, b % per, (int)(b / per), lds);
}

template <typename T, int D>
void launch_d(const AttendParams &p, const AttendParams &q, int KT, hipStream_t st) {
    const unsigned grid = (unsigned)(p.units * p.Hkv * p.S + q.units * q.Hkv * q.S);
    constexpr int NT = prompt_waves<T, D>() * SSA_WAVE;
    if (KT == 32) cache_prompt_kernel<T, D, 32><<<grid, NT, 0, st>>>(p, q.units, q.S, q.chunk, q.part_ml, q.part_o);
    else cache_prompt_kernel<T, D, 64><<<grid, NT, 0, st>>>(p, q.units, q.S, q.chunk, q.part_ml, q.part_o);
}

template <typename T>
void launch_t(const AttendParams &p, const AttendParams &q, int D, int KT, hipStream_t st) {
    if (D == 64) launch_d<T, 64>(p, q, KT, st);
    else if (D == 128) launch_d<T, 128>(p, q, KT, st);
    else launch_d<T, 256>(p, q, KT, st);
}

}  // namespace

int ssa_cache_prompt_columns(int dtype, int D) {
    return 16 * (dtype == SSA_F32 && D == 256 ? prompt_waves<float, 256>() : prompt_waves<bf16_t, 128>());
}

void ssa_cache_prompt_launch(const AttendParams &p, const AttendParams &q, int dtype, int D, int KT,
                             hipStream_t st) {
    if (dtype == SSA_F32) launch_t<float>(p, q, D, KT, st);
    else if (dtype == SSA_BF16) launch_t<bf16_t>(p, q, D, KT, st);
    else launch_t<f16_t>(p, q, D, KT, st);
}
