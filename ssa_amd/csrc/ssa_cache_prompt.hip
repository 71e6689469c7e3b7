// ssa_cache_prompt.hip -- attention over the paged 8-bit cache for many query rows
// of one request (prompts and their chunks).
//
// The products and the mapping of keys to lanes are those of ssa_cache_attend.hip
// (S^T = K Q^T, O^T = V^T P^T, a column is a query row, P^T stays in registers).
// Here each wave owns 16 RT columns and walks every key tile of the workgroup's
// range, so the tiles are shared: the waves convert a tile's codes to 16-bit floats
// once, into LDS, in the order in which the matrix operands read them (a fragment is
// 64 slots of 16 bytes: every LDS access is free of conflicts), double-buffered, with the next tile's codes already on their way from memory.  Bound by the matrix
// pipe and the exponentials together.
#include "ssa_cache_attend_dev.h"

namespace {

// 16-byte pieces of LDS a workgroup uses
template <int D, int KT> constexpr int prompt_lds() {
    return 2 * 2 * (KT / 16 * (D / 64) + D / 16 * (KT / 32) / 2) * SSA_WAVE + 1;
}

template <typename T, int D, int KT, int RT>
__device__ __forceinline__ void prompt_unit(const AttendParams &p, unsigned block, int split, u32x4 *lds) {
    typedef Columns<T, D, KT, RT> C;
    typedef typename C::QV QV;
    typedef typename C::PV PV;
    constexpr int NQ = C::NQ, NP = C::NP, NB = C::NB, DP = C::DP, ND = C::ND, KS = C::KS;
    constexpr int CT = ATT_WAVES * 16 * RT;
    // a load unit: 16 codes a lane, two fragments
    constexpr int KU = NB * DP, VU = ND * KS / 2, NU = KU + VU, UW = NU / ATT_WAVES;
    u32x4 (*frag)[2 * NU][SSA_WAVE] = (u32x4 (*)[2 * NU][SSA_WAVE])lds;    // two buffers
    int *most_lds = (int *)(lds + prompt_lds<D, KT>() - 1);

    const int lane = lane_id(), lrow = lane >> 2, lpiece = lane & 3;
    const int to = slot_of(lrow, lpiece), from = slot_of(lane & 15, lane >> 4);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / SSA_WAVE);
    // kv heads run fastest: an XCD's workgroups share their heads' pages in its L2;
    // units run backwards, those with the most keys first
    const int h = (int)(block % (unsigned)p.Hkv);
    const int u = p.units - 1 - (int)(block / (unsigned)p.Hkv);
    Unit un;
    if (!locate_unit(p, u, CT, un)) return;
    const int wc0 = un.c0 + wave * 16 * RT;   // this wave's first column
    C w;
    w.start(p, un, wc0, un.c1, h);
    if (lane == 0) most_lds[wave] = w.most;
    __syncthreads();
    int most_wg = -1;
#pragma unroll
    for (int i = 0; i < ATT_WAVES; ++i) most_wg = max(most_wg, most_lds[i]);
    most_wg = __builtin_amdgcn_readfirstlane(most_wg);

    const int page = 1 << p.page_shift;
    const int n_tiles = most_wg < 0 ? 0 : most_wg / KT + 1;
    const int tile0 = split * p.chunk, tile1 = min(tile0 + p.chunk, n_tiles);
    const int sub_shift = p.page_shift - (KT == 64 ? 6 : 5);
    const int32_t *table = p.table + (int64_t)(un.req < 0 ? 0 : un.req) * p.table_stride;

    // this wave's load units: key block b, columns 64 i.. ; or value rows
    int off[UW];
    u32x4 raw[UW];
#pragma unroll
    for (int x = 0; x < UW; ++x) {
        const int un_ = wave * UW + x;
        if (un_ < KU) {
            const int b = un_ / DP, i = un_ % DP;
            off[x] = (KT / 4 * (lrow >> 2) + 4 * b + (lrow & 3)) * D + i * 64 + lpiece * 16;
        } else {
            const int i = un_ - KU;
            off[x] = KT == 64 ? ((i * 16 + lrow) << p.page_shift) + 16 * lpiece
                              : ((i * 32 + lrow) << p.page_shift) + 8 * lpiece;
        }
    }
    struct Tile { int pg; float ks, vs; };
    // A tile's table entry is loaded a tile ahead of its codes, whatever it is (of the
    // last tile, past the end), and judged where they are: nothing waits for it.
    const int last_entry = (max(tile1, 1) - 1) >> sub_shift;
    auto entry = [&](int tile) { return table[min(tile >> sub_shift, last_entry)]; };
    auto fetch = [&](int tile, int pg, Tile &ti) {
        ti.pg = tile < tile1 && pg >= 0 && pg < p.num_pages ? pg : -1;
        if (ti.pg < 0) return;
        const int sub = tile & ((1 << sub_shift) - 1);
        const int64_t ph = (int64_t)pg * p.Hkv + h;
        ti.ks = p.ks[ph];
        ti.vs = p.vs[ph];
        const uint8_t *kb = p.k + ph * D * page + sub * KT * D;
        const uint8_t *vb = p.v + ph * D * page + sub * KT;
#pragma unroll
        for (int x = 0; x < UW; ++x) {
            if (wave * UW + x < KU) {
                raw[x] = *(const u32x4 *)(kb + off[x]);
            } else if (KT == 64) {
                raw[x] = *(const u32x4 *)(vb + off[x]);
            } else {
                const u32x2 a = *(const u32x2 *)(vb + off[x]);
                const u32x2 b = *(const u32x2 *)(vb + off[x] + (16 << p.page_shift));
                raw[x] = u32x4{a.x, a.y, b.x, b.y};
            }
        }
    };
    auto stage = [&](int buf, const Tile &ti) {
        if (ti.pg < 0) return;
#pragma unroll
        for (int x = 0; x < UW; ++x) {
            const int f = 2 * (wave * UW + x);
            if (wave * UW + x < KU) {
                *(QV *)&frag[buf][f][to] = Ops<T>::key(raw[x].x, raw[x].y);
                *(QV *)&frag[buf][f + 1][to] = Ops<T>::key(raw[x].z, raw[x].w);
            } else {
                *(PV *)&frag[buf][f][to] = Ops<T>::value(raw[x].x, raw[x].y, ti.vs);
                *(PV *)&frag[buf][f + 1][to] = Ops<T>::value(raw[x].z, raw[x].w, ti.vs);
            }
        }
    };

    Tile cur{-1, 0.f, 0.f}, nxt{-1, 0.f, 0.f};
    int pg2 = -1;
    if (tile0 < tile1) {
        const int pg0 = entry(tile0), pg1 = entry(tile0 + 1);
        pg2 = entry(tile0 + 2);
        fetch(tile0, pg0, cur);
        stage(0, cur);
        fetch(tile0 + 1, pg1, nxt);
    }
    __syncthreads();
    for (int tile = tile0; tile < tile1; ++tile) {
        const int buf = (tile - tile0) & 1;
        stage(buf ^ 1, nxt);
        Tile nn{-1, 0.f, 0.f};
        fetch(tile + 2, pg2, nn);
        pg2 = entry(tile + 3);
        const int key0 = tile * KT;
        if (cur.pg >= 0 && key0 <= w.most) {
            f32x4 s[RT][NB];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int b = 0; b < NB; ++b) s[rt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
            // fragments are read a group ahead of the products that take them, the
            // first values' during the softmax
            constexpr int KG = DP * 2, VG = ND > 2 ? 2 : ND;
            const u32x4 *kl = &frag[buf][0][from], *vl = &frag[buf][2 * KU][from];
            u32x4 kf[2][KG], vf[2][VG * KS];
#pragma unroll
            for (int k = 0; k < KG; ++k) kf[0][k] = kl[k * SSA_WAVE];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b + 1 < NB) {
#pragma unroll
                    for (int k = 0; k < KG; ++k) kf[(b + 1) & 1][k] = kl[((b + 1) * KG + k) * SSA_WAVE];
                } else {
#pragma unroll
                    for (int k = 0; k < VG * KS; ++k) vf[0][k] = vl[k * SSA_WAVE];
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < KG; ++k)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int n = NQ - 1; n >= 0; --n)
                            s[rt][b] = mfma(__builtin_bit_cast(QV, kf[b & 1][k]), w.q[rt][k][n], s[rt][b]);
            }
            PV pf[RT][KS][NP];
            w.softmax(s, cur.ks, cur.vs, key0, pf);
#pragma unroll
            for (int i = 0; i < ND / VG; ++i) {
                if (i + 1 < ND / VG)
#pragma unroll
                    for (int k = 0; k < VG * KS; ++k)
                        vf[(i + 1) & 1][k] = vl[((i + 1) * VG * KS + k) * SSA_WAVE];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < VG; ++j)
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int n = NP - 1; n >= 0; --n)
                                w.o[rt][i * VG + j] = mfma(__builtin_bit_cast(PV, vf[i & 1][j * KS + k]),
                                                           pf[rt][k][n], w.o[rt][i * VG + j]);
            }
        }
        __syncthreads();
        cur = nxt;
        nxt = nn;
    }
    w.finish(p, un, wc0, un.c1, h, split, tile0 < tile1);
}

// Both kinds of units in one launch: requests with few columns (p, first) and with
// many (q); their lengths, and so which there are, are known on the GPU alone.
template <typename T, int D, int KT, int RT>
__global__ void __launch_bounds__(ATT_WAVES * SSA_WAVE, D <= 128 ? 2 : 1)
cache_mixed_kernel(AttendParams p, AttendParams q) {
    constexpr int A = attend_lds<D, KT, 1, true>(), B = prompt_lds<D, KT>();
    __shared__ u32x4 lds[A > B ? A : B];
    const unsigned pu = (unsigned)(p.units * p.Hkv), few = pu * (unsigned)p.S;
    if (blockIdx.x < few) {
        attend_unit<T, D, KT, 1, true>(p, blockIdx.x % pu, (int)(blockIdx.x / pu), lds);
    } else {
        const unsigned b = blockIdx.x - few, qu = (unsigned)(q.units * q.Hkv);
        prompt_unit<T, D, KT, RT>(q, b % qu, (int)(b / qu), lds);
    }
}

// Most 16-column tiles of a wave: as many as the registers hold beside O (RT D / 4),
// the scores and the queries.
template <typename T, int D> constexpr int max_rt() {
    return sizeof(T) == 4 ? (D <= 64 ? 2 : 1) : (D <= 64 ? 4 : (D <= 128 ? 2 : 1));
}

template <typename T, int D, int RT>
void launch_rt(const AttendParams &p, const AttendParams &q, int KT, hipStream_t st) {
    const unsigned grid = (unsigned)(p.units * p.Hkv * p.S + q.units * q.Hkv * q.S);
    if (KT == 32) cache_mixed_kernel<T, D, 32, RT><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p, q);
    else cache_mixed_kernel<T, D, 64, RT><<<grid, ATT_WAVES * SSA_WAVE, 0, st>>>(p, q);
}

template <typename T, int D>
void launch_d(const AttendParams &p, const AttendParams &q, int KT, int RT, hipStream_t st) {
    constexpr int M = max_rt<T, D>();
    if constexpr (M >= 4)
        if (RT == 4) return launch_rt<T, D, 4>(p, q, KT, st);
    if constexpr (M >= 2)
        if (RT == 2) return launch_rt<T, D, 2>(p, q, KT, st);
    launch_rt<T, D, 1>(p, q, KT, st);
}

template <typename T>
void launch_t(const AttendParams &p, const AttendParams &q, int D, int KT, int RT, hipStream_t st) {
    if (D == 64) launch_d<T, 64>(p, q, KT, RT, st);
    else if (D == 128) launch_d<T, 128>(p, q, KT, RT, st);
    else launch_d<T, 256>(p, q, KT, RT, st);
}

}  // namespace

int ssa_cache_prompt_max_rt(int dtype, int D) {
    if (dtype == SSA_F32)
        return D == 64 ? max_rt<float, 64>() : (D == 128 ? max_rt<float, 128>() : max_rt<float, 256>());
    return D == 64 ? max_rt<bf16_t, 64>() : (D == 128 ? max_rt<bf16_t, 128>() : max_rt<bf16_t, 256>());
}

void ssa_cache_mixed_launch(const AttendParams &p, const AttendParams &q, int dtype, int D, int KT,
                            int RT, hipStream_t st) {
    if (dtype == SSA_F32) launch_t<float>(p, q, D, KT, RT, st);
    else if (dtype == SSA_BF16) launch_t<bf16_t>(p, q, D, KT, RT, st);
    else launch_t<f16_t>(p, q, D, KT, RT, st);
}
