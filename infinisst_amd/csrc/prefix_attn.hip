// Attention of a batch whose sequences share one long prefix in front of keys of their own (gfx950).
//
// Row t of the n rows of sequence b sees the P prefix keys and its own keys j < len_b - n + t + 1:
//     o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)   over both sets, for any m that keeps the exponentials in range (m: the column's reference).
// One launch computes partial (O, m, l) triples, a second one joins them.  A workgroup of the first launch takes one of two roles:
//   block: 32 NW columns ((row, head) pairs of one key head, over ALL sequences) against a span of the prefix, or the columns of one sequence against its own keys.  Every tile of 32 keys
//          goes through LDS once for all columns.  Bound by the matrix instructions and what goes with them.
//   span:  16 NQ columns of ONE sequence against its own keys (or of the whole batch against the prefix where it has no more columns than that); the waves split the keys.  Bound by the read.
// Scores are computed transposed, S^T = K Q^T, so that a lane holds one column: statistics and rescaling are per lane, and the exponentials are already in the layout the value product
// O^T = V^T P^T wants its B operand in (the order of the keys inside a 16- or 32-key step is free as long as V^T is read in the same order: two transposed LDS reads).
// The weights enter the value product as bf16 (off by 2^-8 relative at most, as the output's own rounding is) and their sum is taken of the rounded ones, so that they still add up to one: bf16
// matrix instructions want both operands so, and a pair of bf16 numbers a weight would double that product.  Over a row's norm the outputs are off by 0.0020 to 0.0024, by 0.0017 from their own rounding
// alone.  Scores, references, sums and accumulators are fp32.
// Measured, 32 heads over 8 key heads of 128: 64 sequences x 16 rows over 8192 shared keys 143 us a call, the first launch 131 = 1048 TFLOP/s (a large matrix product of the library reaches 1192 on the
// same card); 64 x 1 row over 1000 own keys 47 us = 5.5 TB/s (a large copy: 4.9, counted both ways).
#include "../../include/infinisst_hip.h"
#include "common.h"
#include "kernels.h"

#include <type_traits>

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((address_space(3))) void* lds_ptr;

#define PA_NW 4                  // waves of a workgroup, two workgroups a CU: the waits of one hide behind the other (eight waves, one a CU: 64 x 16 rows 151 -> 158 us, 64 x 5 rows 78 -> 92)
#define PA_TILE 32               // keys of a block tile
#define PA_HEAD 16.f             // octaves by which a column's reference stands above the maximum that set it
#define PA_RAISE 1.f             // sum of a lane's weights in a step from which a column's reference is raised

// [first, first + n) = the rows of sequence b, clipped to the launch's rows
__device__ __forceinline__ void seq_rows(const isst_prefix_attn& a, int b, int& first, int& n) {
    if (a.row_starts) {
        first = min(max(a.row_starts[b], 0), a.rows);
        n = max(min(max(a.row_starts[b + 1], 0), a.rows) - first, 0);
    } else {
        n = a.rows / a.seqs;
        first = b * n;
    }
}
// the sequence that owns `row` (-1: none): the last one that starts at or before it
__device__ __forceinline__ int seq_of_row(const isst_prefix_attn& a, int row) {
    if (!a.row_starts) return row / (a.rows / a.seqs);
    int lo = 0, hi = a.seqs;  // row_starts[lo - 1] <= row < row_starts[hi]
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.row_starts[mid] <= row) lo = mid + 1; else hi = mid;
    }
    return lo > 0 && row < a.row_starts[lo] ? lo - 1 : -1;
}

struct PrefixPlan {
    unsigned magic;                              // ceil(2^32 / G), 0 for G = 1 (group_of)
    int prefix_block, prefix_tiles, prefix_splits, prefix_units;  // block form or span form; column tiles, key spans; units padded to a multiple of 8
    int own_block, own_tiles, own_splits, own_units;                           // column tiles of a sequence (a longer one walks on), key spans
    int slots;
    float* o;                                    // [slots][rows * heads][D] fp32, unnormalised
    float2* ml;                                  // [slots][rows * heads]: reference (in units of log2), sum
};
// x / G for a column counted from the start of a row (x < G + 128, G < 2^15: exact)
__device__ __forceinline__ int group_of(int x, unsigned magic) { return magic ? (int)__umulhi((unsigned)x, magic) : x; }
// what a workgroup attends to: columns c0 .. ncols - 1 of a sequence (column c = its row c / G, head kvh G + c % G) over `keys` keys; column c sees keys j < limit0 + c / G where causal
struct KeySpan {
    const bf16_t *k, *v;
    long kstride, vstride;
    int keys, first, ncols, kvh;
    bool causal;
    int limit0;
};
__device__ __forceinline__ int sees(const KeySpan& s, int t) { return s.causal ? min(max(s.limit0 + t, 0), s.keys) : s.keys; }

// XOR swizzle of the 16-byte chunks of a K / V tile row: 16 rows read at one chunk (K fragments) and 4 rows x 4 chunks (transposed V reads) both cover all 64 banks once
template <int D>
__device__ __forceinline__ int tile_off(int row, int ch) {
    if constexpr (D == 128) return 256 * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3)));
    return 128 * row + 16 * (ch ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)));
}
__device__ __forceinline__ u32x2_t read_tr(const char* p) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)p));
}
// LDS-DMA from a buffer descriptor at a tile's first row (a lane's offset and the scalar one of its row group together stay below 2^32).  As global loads the compiler would count it as an LDS
// access that ends in no known order, and wait for ALL fragments in front of the first product: 64 sequences x 16 rows over 8192 keys 168 us, so 160.  (The span role waits for all of a step anyway,
// and takes global loads: 64 x 1 row 49 us with descriptors, 47 without.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* p) { return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0xffffffffu, 0x00020000); }
__device__ __forceinline__ void dma(const __amdgpu_buffer_rsrc_t& r, char* dst, unsigned lane_offset, unsigned rows_offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)dst, 16, lane_offset, rows_offset, 0, 0);
}

// Keys [lo, hi) of one column added to its stored partial result, whose reference covers them.  Only for tiles that hold inf or NaN values and that some column of a wave does not see
// whole: in a matrix product 0 x inf would reach the columns that do not see the key.
template <int D>
__device__ void add_keys(const isst_prefix_attn& a, const PrefixPlan& p, const KeySpan& w, int slot, int c, int lo, int hi) {
    const int G = a.heads / a.kv_heads, t = c / G, head = w.kvh * G + c % G;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const long at = (long)slot * a.rows * a.heads + (long)(w.first + t) * a.heads + head;
    const float m = p.ml[at].x, neg = m == -INFINITY ? 0.f : -m;
    const bf16_t* q = a.q + (w.first + t) * a.q_row + head * a.q_head;
    hi = min(hi, sees(w, t));
    for (int j = lo; j < hi; ++j) {
        float s = 0.f;
        for (int d = lane; d < D; d += 64) s += bf2f(q[d]) * bf2f(w.k[j * w.kstride + d]);
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(wave_sum(s), a.scale * 1.44269504088896340736f, neg));
        for (int d = lane; d < D; d += 64) p.o[at * D + d] += e * bf2f(w.v[j * w.vstride + d]);
    }
}

// ---------------------------------------------------------------------------------------------------------------- block role
// columns [c0, c0 + 32 NW) against the key tiles of span `split` of `splits`.  A wave owns 32 columns.  Key and value tiles arrive by LDS-DMA in rings of four stages (64 KB: two workgroups a
// CU), two tiles between barriers.  The matrix instructions of a tile are 512 cycles of the matrix pipe, its vector instructions 315 cycles of issue: one after the other the two waves of a
// SIMD take 184 us for 64 x 16 rows over 8192 keys, join included (tiles through registers or by LDS-DMA, one a barrier); with the exponentials between the matrix instructions of the neighbouring
// tiles 176; two tiles a barrier and no 64-bit address arithmetic per tile 166; fragment waits counted 160; the ring's stages as constants 157.  (All of these on a chip that 20 calls
// do not bring to its clock; in the long run the last form takes 143.)  The matrix pipe is busy 56 % of the time that a workgroup runs; the waves wait for it or for each other's.
template <int D, int NW>
__device__ __forceinline__ void block_role(const isst_prefix_attn& a, const PrefixPlan& p, char* lds, const KeySpan& w, int c0, int split, int splits, int slot) {
    constexpr int ROWB = 2 * D, CH = D / 8, LOADS = PA_TILE * CH / (NW * 64), RSTEP = NW * 64 / CH, QS = D / 16, DT = D / 32, STAGE = PA_TILE * ROWB;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, half = lane >> 5;
    const int G = a.heads / a.kv_heads, cw = c0 + 32 * wave;
    const int total = (sees(w, (min(c0 + 32 * NW, w.ncols) - 1) / G) + PA_TILE - 1) / PA_TILE, per = (total + splits - 1) / splits, tile0 = split * per, tiles = min(per, total - tile0);
    const bool wave_live = cw < w.ncols, live = cw + c32 < w.ncols;
    const int t0 = cw / G, x = cw % G + c32, t = live ? t0 + group_of(x, p.magic) : t0;
    const int head = w.kvh * G + (live ? x - (t - t0) * G : 0);
    const int limit = live ? sees(w, t) : w.keys, see_least = sees(w, t0), see_most = wave_live ? sees(w, (min(cw + 32, w.ncols) - 1) / G) : 0;
    const int mine = min(tiles, (see_most + PA_TILE - 1) / PA_TILE - tile0);  // tiles that this wave's columns see

    u32x4_t qf[QS];
#pragma unroll
    for (int s = 0; s < QS; ++s)
        qf[s] = live ? *reinterpret_cast<const u32x4_t*>(a.q + (w.first + t) * a.q_row + head * a.q_head + 16 * s + 8 * half) : (u32x4_t){0u, 0u, 0u, 0u};
    // keys of tile i go to key stage i % 4, its values to value stage i % 4, by LDS-DMA: a wave fills 1 KB at a time in lane order, so the swizzle is in which chunk of its row a lane asks
    // for.  Rows behind the last key repeat it.
    const int lr = tid / CH, lc = tile_off<D>(lr, tid % CH) % ROWB;
    const unsigned krows = RSTEP * 2 * (unsigned)w.kstride, vrows = RSTEP * 2 * (unsigned)w.vstride;  // bytes between the rows of two loads
    const unsigned koff = lr * (int)(2 * w.kstride) + lc, voff = lr * (int)(2 * w.vstride) + lc;
    char *const kring = lds, *const vring = lds + 4 * STAGE;
    auto stage = [&](int i) { return (i & 3) * STAGE; };
    auto fetch = [&](const bf16_t* rows0, long stride, int i, char* stage) {
        const int left = w.keys - (tile0 + i) * PA_TILE;
        if (i >= tiles) return;
        const __amdgpu_buffer_rsrc_t src = rows_at(rows0 + (tile0 + i) * PA_TILE * stride);
#pragma unroll
        for (int k = 0; k < LOADS; ++k)
            dma(src, stage + (k * NW + wave) * 1024, min(lr + k * RSTEP, left - 1) * (int)(2 * stride) + lc, 0);
    };
    fetch(w.k, w.kstride, 0, kring);
    fetch(w.k, w.kstride, 1, kring + STAGE);
    fetch(w.k, w.kstride, 2, kring + 2 * STAGE);
    fetch(w.v, w.vstride, 0, vring);
    f32x16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    unsigned ill_tiles = 0;
    const float c2 = a.scale * 1.44269504088896340736f;  // exp(scale s - ..) = exp2(c2 s - ..)

    // everything asked for has landed, for every wave, and every wave is done with what it read
    auto turn = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    turn();
    // LDS offsets of a lane inside its stage; other product steps and columns are an XOR away (the swizzle is one), other rows a constant
    const int klane = tile_off<D>(c32, half), vlane = tile_off<D>(4 * half + ((lane >> 2) & 3), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
    auto key_frag = [&](const char* kst, int s) { return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(kst + (klane ^ 32 * s))); };
    // 16 keys a product: slots j < 4 of half h = keys 16 k + 4 h + j, j >= 4 = keys 16 k + 8 + 4 h + (j - 4)
    auto value_frag = [&](const char* vst, int k, int d) {
        const u32x2_t v1 = read_tr(vst + (vlane ^ 64 * d) + 16 * k * ROWB), v2 = read_tr(vst + (vlane ^ (64 * d + 32)) + (16 * k + 8) * ROWB);
        return __builtin_bit_cast(bf16x8_t, (u32x4_t){v1.x, v1.y, v2.x, v2.y});
    };
    auto scores = [&](const char* kst) {
        f32x16_t sc;
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
        for (int s = 0; s < QS; ++s) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key_frag(kst, s), __builtin_bit_cast(bf16x8_t, qf[s]), sc, 0, 0, 0);
        return sc;
    };
    f32x16_t sc = scores(kring);  // (no tile: of whatever the stage holds, unused -- as behind the last tile below)
    turn();                       // (keys 4 take the place of keys 0)
    // m becomes the maximum of what it covers and of these scores, and PA_HEAD
    auto raise = [&]() {
        float mx = sc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sc[r]);
        mx = __builtin_fmaf(fmaxf(mx, __shfl_xor(mx, 32, WAVE)), c2, PA_HEAD);
        const float m2 = fmaxf(m, mx), keep = m == m2 ? 1.f : m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m2);
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] *= keep;
        m = m2;
    };
    // weights of the tile (bf16 pairs in the layout of the value product) and their sum in this lane, as the product will see them
    auto weights = [&](u32x4_t (&pf)[2], float neg) {
        const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = 8 * k + 2 * q;
                const uint32_t pair = pack_bf(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[r], c2, neg)), __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r + 1], c2, neg)));
                pf[k][q] = pair;
                sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), one, sum, false);
            }
        return sum;
    };
    // Step i: the scores of tile i are in sc and become weights; on the way the values of tile i - 1, whose weights are in pf, are added and the scores of tile i + 1 are computed.
    // A column's reference m stands 16 octaves above the maximum of its first tile (and of its edge tiles): weights are exponentials against it, bf16 and fp32 lose no bit by their size, so other
    // maxima are not looked for -- that and the running sum were 100 of the 169 vector instructions of a tile -- and only weights whose sum in a lane passes one (or is NaN) move m, before
    // anything of the tile was used.  A weight that is used is at most one, as with a running maximum: the accumulators hold whatever sum |v| over the keys does.  Scores have to rise by 11
    // above a column's first tile to move m.  (A reference at the maximum itself and weights up to 2^16 took the same time, and values above 2^111 overflowed.)
    u32x4_t pf[2];
    enum { NONE, WHOLE, EDGE } before = NONE;  // what tile i - 1 was: EDGE, some column did not see some key of it
    auto ref = [&]() { return m == -INFINITY ? 0.f : -m; };
    auto add_values = [&](int i) {  // of tile i
        if (before == EDGE) {
            bool ill = false;  // inf or NaN among the values: they are added behind the loop
#pragma unroll 1
            for (int k = 0; k < PA_TILE * ROWB / 1024; ++k) {
                const u32x4_t v = *reinterpret_cast<const u32x4_t*>(vring + (i & 3) * STAGE + 1024 * k + 16 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) ill |= (v[e] & 0x7f80u) == 0x7f80u || (v[e] & 0x7f800000u) == 0x7f800000u;
            }
            if (__any(ill)) {
                ill_tiles |= 1u << min((tile0 + i) - see_least / PA_TILE, 31);
                return;
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_frag(vring + (i & 3) * STAGE, k, d), __builtin_bit_cast(bf16x8_t, pf[k]), o[d], 0, 0, 0);
    };
    // the first tile and those at the edge: one thing after the other
    auto slow_step = [&](int i, bool edge) {
        if (before != NONE) add_values(i - 1);
        if (edge) {
            const int lim = limit - (tile0 + i) * PA_TILE - 4 * half;
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((r & 3) + 8 * (r >> 2) >= lim) sc[r] = -INFINITY;
        }
        raise();
        l += weights(pf, ref());
        before = edge ? EDGE : WHOLE;
        sc = scores(kring + stage(i + 1));
    };
    // the others: matrix and vector instructions in turn, since the two waves of a SIMD do not find enough of the other's kind by themselves
    auto step = [&](const char* __restrict__ kst, const char* __restrict__ vst) {
        bf16x8_t kf[QS], vf[2][DT];
#pragma unroll
        for (int s = 0; s < QS / 2; ++s) kf[s] = key_frag(kst, s);
#pragma unroll
        for (int d = 0; d < DT; ++d) vf[0][d] = value_frag(vst, 0, d);
        __builtin_amdgcn_sched_barrier(0);
        const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
        f32x16_t sn;
#pragma unroll
        for (int r = 0; r < 16; ++r) sn[r] = 0.f;
        u32x4_t pn[2];
        float sum = 0.f;
        constexpr int EVERY = 8 / QS;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const int q = c / EVERY;
            if (c % EVERY == 0) {
                sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[q], __builtin_bit_cast(bf16x8_t, qf[q]), sn, 0, 0, 0);
                if (q < QS / 2) kf[q + QS / 2] = key_frag(kst, q + QS / 2);
            }
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * c], c2, -m)), e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * c + 1], c2, -m));
            if (c % EVERY == 0) {
                o[q % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[q / DT][q % DT], __builtin_bit_cast(bf16x8_t, pf[q / DT]), o[q % DT], 0, 0, 0);
                if (q < DT) vf[1][q] = value_frag(vst, 1, q);
            }
            const uint32_t pair = pack_bf(e0, e1);
            pn[c / 4][c % 4] = pair;
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), one, sum, false);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__any(!(sum <= PA_RAISE))) {  // (no reference yet, all scores so far -inf: weights of inf or NaN, which set one)
            raise();
            sum = weights(pn, ref());
        }
        l += sum;
        pf[0] = pn[0]; pf[1] = pn[1];
        sc = sn;
    };
    const int whole = min(mine, see_least / PA_TILE - tile0);  // tiles that every column of the wave sees whole
    // Two tiles between barriers: keys i + 1, i + 2 and values i - 1, i are read while keys i + 3, i + 4 and values i + 1, i + 2 arrive
    const char *ksrc = reinterpret_cast<const char*>(w.k + (tile0 + 3) * PA_TILE * w.kstride), *vsrc = reinterpret_cast<const char*>(w.v + (tile0 + 1) * PA_TILE * w.vstride);
    auto ask = [&](int i, char* __restrict__ knew0, char* __restrict__ knew1, char* __restrict__ vnew0, char* __restrict__ vnew1) {
        if (i + 5 < tiles) {
            const __amdgpu_buffer_rsrc_t kr = rows_at(ksrc), vr = rows_at(vsrc);
#pragma unroll
            for (int k = 0; k < LOADS; ++k) {
                dma(kr, knew0 + (k * NW + wave) * 1024, koff, k * krows);
                dma(kr, knew1 + (k * NW + wave) * 1024, koff, (k + LOADS) * krows);
                dma(vr, vnew0 + (k * NW + wave) * 1024, voff, k * vrows);
                dma(vr, vnew1 + (k * NW + wave) * 1024, voff, (k + LOADS) * vrows);
            }
            ksrc += 2l * LOADS * krows;
            vsrc += 2l * LOADS * vrows;
        } else {
            fetch(w.k, w.kstride, i + 3, knew0);
            fetch(w.k, w.kstride, i + 4, knew1);
            fetch(w.v, w.vstride, i + 1, vnew0);
            fetch(w.v, w.vstride, i + 2, vnew1);
        }
    };
    auto two_steps = [&](int i, char* __restrict__ knew0, char* __restrict__ knew1, char* __restrict__ vnew0, char* __restrict__ vnew1, const char* __restrict__ kst0,
                         const char* __restrict__ kst1, const char* __restrict__ vst0, const char* __restrict__ vst1) {
        ask(i, knew0, knew1, vnew0, vnew1);
        step(kst0, vst0);
        step(kst1, vst1);
        turn();
    };
    int i = 0;
    while (i < ((tiles + 1) & ~1)) {
        if (!(i & 1)) ask(i, kring + stage(i + 3), kring + stage(i), vring + stage(i + 1), vring + stage(i + 2));
        if (i < mine) slow_step(i, i >= whole);
        else if (before != NONE) {
            add_values(i - 1);
            before = NONE;
        }
        if (i & 1) turn();
        ++i;
        if (!(i & 1)) {
            auto at = [&](int i, int r) {  // r = i mod 4
                two_steps(i, kring + stage(r + 3), kring + stage(r), vring + stage(r + 1), vring + stage(r + 2), kring + stage(r + 1), kring + stage(r + 2), vring + stage(r + 3), vring + stage(r));
            };
            while (i + 1 < whole) {
                if (i & 2) {
                    at(i, 2);
                    i += 2;
                    if (i + 1 >= whole) break;
                }
                at(i, 0);
                i += 2;
            }
        }
    }
    if (before != NONE) add_values(mine - 1);
    __syncthreads();  // (the last values are read behind the last turn)
    // ---- (m, l) and the accumulators; these turn through the wave's part of LDS so that whole rows of D floats are stored ----
    int jl = lane;
    asm volatile("" : "+v"(jl));
    l += __shfl_xor(l, 32, WAVE);
    const long base = (long)slot * a.rows * a.heads;
    if (live && half == 0) p.ml[base + (long)(w.first + t) * a.heads + head] = make_float2(m, l);
    if (tiles <= 0 || !wave_live) return;  // (uniform per wave; l = 0 tells the join that there is nothing to read)
    float* red = reinterpret_cast<float*>(lds) + wave * (32 * D);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d4 = 8 * d + 2 * r4 + (jl >> 5), c = jl & 31;
            *reinterpret_cast<f32x4_t*>(red + c * D + 4 * (d4 ^ (c & (D / 4 - 1)))) = (f32x4_t){o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
        }
    __builtin_amdgcn_wave_barrier();
    constexpr int L4 = D / 4, CPI = 64 / L4;
    const int d4 = jl % L4;
    for (int c = jl / L4; c < 32; c += CPI) {
        if (cw + c >= w.ncols) break;
        const int xc = cw % G + c, tc = group_of(xc, p.magic);
        const long at = base + (long)(w.first + t0 + tc) * a.heads + w.kvh * G + (xc - tc * G);
        *reinterpret_cast<f32x4_t*>(p.o + at * D + 4 * d4) = *reinterpret_cast<const f32x4_t*>(red + c * D + 4 * (d4 ^ (c & (L4 - 1))));
    }
    if (ill_tiles) {
        __threadfence_block();
        for (int c = 0; c < 32 && cw + c < w.ncols; ++c)
            for (int k = 0; k < 32; ++k)
                if (ill_tiles >> k & 1) {
                    const int j = (see_least / PA_TILE + k) * PA_TILE;
                    add_keys<D>(a, p, w, slot, cw + c, j, j + PA_TILE);
                }
    }
}

// ---------------------------------------------------------------------------------------------------------------- span role
// columns [c0, c0 + 16 NQ) over all their keys; the waves of `splits` workgroups take 32 keys at a time each and are joined at the end.  A step's keys and values arrive by LDS-DMA in a buffer of
// the wave's own (no barrier), go to registers in one piece, and the next step's are asked for before the first product.  64 x 1 row over 1000 own keys: 5.5 TB/s.  (Keys straight to registers in
// the layout of the product, values in two buffers: 64 x 5 rows 84 -> 82.5 us, 64 x 1 row 46.6 -> 46.0, but 33 x 1..3 rows with heads of 64 16.3 -> 17.3.)
template <int D, int NW, int NQ>
__device__ __forceinline__ void span_role(const isst_prefix_attn& a, const PrefixPlan& p, char* lds, const KeySpan& w, int c0, int split, int splits, int slot) {
    constexpr int ROWB = 2 * D, CH = D / 8, VL = 32 * CH / 64, VR = 64 / CH, QS = D / 32, NT = D / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int G = a.heads / a.kv_heads, t0 = c0 / G, x0 = c0 % G;
    const int see_least = sees(w, t0), see_most = sees(w, (min(c0 + 16 * NQ, w.ncols) - 1) / G);
    char *const kl = lds + wave * (64 * ROWB), *const vl = kl + 32 * ROWB;  // 32 keys and their values, this wave's alone
    // 1 KB of whole lines an instruction (fragments read from memory are 64 pieces of 16 bytes, a cycle of the L1 cache each); rows behind the last key repeat it
    const int lr = lane / CH;
    auto fetch = [&](const bf16_t* rows0, long stride, int j0, char* dst) {
        const char* src = reinterpret_cast<const char*>(rows0 + j0 * stride);
        const int last = see_most - 1 - j0;
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const int row = lr + i * VR, lc = tile_off<D>(row, lane % CH) % ROWB;
            __builtin_amdgcn_global_load_lds((const void*)(src + (unsigned)(min(row, last) * (int)(2 * stride) + lc)), (lds_ptr)(dst + 1024 * i), 16, 0, 0);
        }
    };
    float2* wml = reinterpret_cast<float2*>(lds + NW * 32 * D * 4);  // [NW][16 NQ], behind the value tiles / turned accumulators
    unsigned& ill_steps = *reinterpret_cast<unsigned*>(wml + NW * 16 * NQ);
    if (tid == 0) ill_steps = 0;
    __syncthreads();
    const int step = 32 * NW * splits;
    int j0 = 32 * (split * NW + wave);
    if (j0 < see_most) {
        fetch(w.k, w.kstride, j0, kl);
        fetch(w.v, w.vstride, j0, vl);
    }

    int limit[NQ];
    u32x4_t qf[NQ][QS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const bool live = c0 + 16 * n + fr < w.ncols;
        const int x = x0 + 16 * n + fr, tc = live ? group_of(x, p.magic) : 0, row = w.first + t0 + tc, head = w.kvh * G + (live ? x - tc * G : 0);
        limit[n] = live ? sees(w, t0 + tc) : w.keys;
#pragma unroll
        for (int s = 0; s < QS; ++s) qf[n][s] = live ? *reinterpret_cast<const u32x4_t*>(a.q + row * a.q_row + head * a.q_head + 32 * s + 8 * fq) : (u32x4_t){0u, 0u, 0u, 0u};
    }
    f32x4_t o[NQ][NT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -INFINITY; l[n] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[n][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    const float c2 = a.scale * 1.44269504088896340736f;
    bool first_step = true;
    for (; j0 < see_most; j0 += step) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        bf16x8_t kf[2][QS], vf[NT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < QS; ++s) kf[t][s] = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(kl + tile_off<D>(16 * t + fr, 4 * s + fq)));
        const int vrow = 4 * fq + ((lane >> 2) & 3), vch = (lane & 3) >> 1, vb8 = 8 * (lane & 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const u32x2_t v1 = read_tr(vl + tile_off<D>(vrow, 2 * t + vch) + vb8), v2 = read_tr(vl + tile_off<D>(16 + vrow, 2 * t + vch) + vb8);
            vf[t] = __builtin_bit_cast(bf16x8_t, (u32x4_t){v1.x, v1.y, v2.x, v2.y});
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (all of the step is in registers: the next one may arrive)
        __builtin_amdgcn_sched_barrier(0);
        if (j0 + step < see_most) {
            fetch(w.k, w.kstride, j0 + step, kl);
            fetch(w.v, w.vstride, j0 + step, vl);
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t sc[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[n][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < QS; ++s) sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][s], __builtin_bit_cast(bf16x8_t, qf[n][s]), sc[n][t], 0, 0, 0);
            }
        const bool edge = j0 + 32 > see_least;  // some column does not see some key of this step
        auto raise = [&]() {  // m becomes the maximum of what it covers and of these scores, and PA_HEAD
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                float mx = sc[n][0][0];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[n][t][r]);
                mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
                mx = __builtin_fmaf(fmaxf(mx, __shfl_xor(mx, 32, WAVE)), c2, PA_HEAD);
                const float m2 = fmaxf(m[n], mx), keep = m[n] == m2 ? 1.f : m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - m2);
                l[n] *= keep;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[n][t][r] *= keep;
                m[n] = m2;
            }
        };
        if (edge) {
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (j0 + 16 * t + 4 * fq + r >= limit[n]) sc[n][t][r] = -INFINITY;
        }
        if (edge || first_step) raise();  // (elsewhere m is a reference, not a maximum: see block_role's step)
        first_step = false;
        u32x4_t pf[NQ];
        float sum[NQ];
        auto weights = [&](float none) {  // none: what a column without a reference subtracts (inf: its weights come out as inf or NaN, and set one)
            const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
            bool over = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const float neg = m[n] == -INFINITY ? none : -m[n];
                sum[n] = 0.f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int t = q >> 1, r = 2 * (q & 1);
                    const uint32_t pair = pack_bf(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][t][r], c2, neg)), __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][t][r + 1], c2, neg)));
                    pf[n][q] = pair;
                    sum[n] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), one, sum[n], false);
                }
                over |= !(sum[n] <= PA_RAISE);
            }
            return __any(over);
        };
        if (weights(INFINITY)) {
            raise();
            (void)weights(0.f);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) l[n] += sum[n];
        if (edge) {
            bool ill = false;  // inf or NaN among the values of a step that not every column sees whole
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4_t v = __builtin_bit_cast(u32x4_t, vf[t]);
#pragma unroll
                for (int w = 0; w < 4; ++w) ill |= (v[w] & 0x7f80u) == 0x7f80u || (v[w] & 0x7f800000u) == 0x7f800000u;
            }
            if (__any(ill)) {  // the step's values are added behind the join
                if (lane == 0) atomicOr(&ill_steps, 1u << min((j0 >> 5) - (see_least >> 5), 31));
                continue;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[t], __builtin_bit_cast(bf16x8_t, pf[n]), o[n][t], 0, 0, 0);
    }
    // ---- join the waves: statistics first, then the weighted accumulators of 16 columns at a time ----
    int jt = tid;
    asm volatile("" : "+v"(jt));  // (keeps this part's addresses out of the registers of the loop above)
    const int jc = jt & 15, jq = (jt & 63) >> 4;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor(l[n], 16, WAVE);
        l[n] += __shfl_xor(l[n], 32, WAVE);
        if (jq == 0) wml[wave * 16 * NQ + 16 * n + jc] = make_float2(m[n], l[n]);
    }
    __syncthreads();  // (also: every wave is done with its value tile, which the accumulators overlay)
    float* red = reinterpret_cast<float*>(lds);  // [NW][16 columns][D]
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, wml[w * 16 * NQ + 16 * n + jc].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 x = wml[w * 16 * NQ + 16 * n + jc];
            L += x.x == -INFINITY ? x.y : x.y * __builtin_amdgcn_exp2f(x.x - M);
        }
        const float keep = m[n] == -INFINITY ? (l[n] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m[n] - M);
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4_t*>(red + (wave * 16 + jc) * D + 16 * t + 4 * (jq ^ (jc & 3))) = o[n][t] * keep;
        __syncthreads();
        for (int e = jt; e < 16 * D / 4; e += NW * 64) {
            const int c = e / (D / 4), d4 = e % (D / 4);
            f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) s += *reinterpret_cast<const f32x4_t*>(red + (w * 16 + c) * D + 4 * ((d4 & ~3) | ((d4 ^ c) & 3)));
            if (c0 + 16 * n + c < w.ncols) {
                const int x = x0 + 16 * n + c, tc = group_of(x, p.magic);
                const long at = (long)slot * a.rows * a.heads + (long)(w.first + t0 + tc) * a.heads + w.kvh * G + (x - tc * G);
                *reinterpret_cast<f32x4_t*>(p.o + at * D + 4 * d4) = s;
            }
        }
        if (wave == 0 && jq == 0 && c0 + 16 * n + jc < w.ncols) {
            const int x = x0 + 16 * n + jc, tc = group_of(x, p.magic);
            p.ml[(long)slot * a.rows * a.heads + (long)(w.first + t0 + tc) * a.heads + w.kvh * G + (x - tc * G)] = make_float2(M, L);
        }
        __syncthreads();
    }
    if (ill_steps && wave == 0)
        for (int c = c0; c < min(c0 + 16 * NQ, w.ncols); ++c)
            for (int k = 0; k < 32; ++k)
                if (ill_steps >> k & 1) add_keys<D>(a, p, w, slot, c, ((see_least >> 5) + k) * 32, ((see_least >> 5) + k) * 32 + 32);
}

template <int D, int NW, int NQ>
__global__ __launch_bounds__(NW * 64, 2) void prefix_attn_partial_kernel(isst_prefix_attn a, PrefixPlan p) {
    constexpr int BLOCK_LDS = 4 * 2 * PA_TILE * 2 * D, SPAN_LDS = NW * 32 * D * 4 + NW * 16 * NQ * 8 + 16;  // (two rings of four stages, or the turned accumulators of a block; the value tiles, or the joined accumulators, and the statistics of a span.  ONE object: with a second one
    // the compiler would wait for every LDS-DMA in front of every read)
    __shared__ __attribute__((aligned(16))) char lds[BLOCK_LDS > SPAN_LDS ? BLOCK_LDS : SPAN_LDS];
    // workgroup i runs on XCD i % 8 (each with an L2 of its own): the column tiles that read the same keys are neighbours on one XCD
    const bool prefix = (int)blockIdx.x < p.prefix_units;
    const int unit = prefix ? blockIdx.x : blockIdx.x - p.prefix_units, G = a.heads / a.kv_heads;
    const int splits = prefix ? p.prefix_splits : p.own_splits, tiles = prefix ? p.prefix_tiles : p.own_tiles;
    const int ct = (unit >> 3) % tiles, g = (unit >> 3) / tiles * 8 + (unit & 7);
    const int kvh = g % a.kv_heads, split = g / a.kv_heads % splits, b = g / a.kv_heads / splits;
    if (b >= (prefix ? 1 : a.seqs)) return;  // (padding)
    KeySpan w;
    int n = a.rows;
    if (prefix) {
        w = {a.k_prefix + kvh * a.kp_head, a.v_prefix + kvh * a.vp_head, a.kp_key, a.vp_key, a.prefix_len, 0, a.rows * G, kvh, false, 0};
    } else {
        int first, len = a.tail_lens[b];
        seq_rows(a, b, first, n);
        first = __builtin_amdgcn_readfirstlane(first);  // (uniform already; a value that the compiler keeps in a vector register would make every key load a loop over lanes)
        n = __builtin_amdgcn_readfirstlane(n);
        len = min(max(__builtin_amdgcn_readfirstlane(len), 0), a.tail_cap);
        w = {a.k_tail + b * a.kt_seq + kvh * a.kt_head, a.v_tail + b * a.vt_seq + kvh * a.vt_head, a.kt_key, a.vt_key, len, first, n * G, kvh, true, len - n + 1};
    }
    const bool block = prefix ? p.prefix_block : p.own_block;
    const int width = block ? 32 * NW : 16 * NQ, slot = prefix ? split : p.prefix_splits + split;
    for (int c0 = ct * width; c0 < w.ncols; c0 += tiles * width) {
        if (c0 != ct * width) __syncthreads();  // (LDS is the last tile's until all are done with it)
        if (block) block_role<D, NW>(a, p, lds, w, c0, split, splits, slot);
        else span_role<D, NW, NQ>(a, p, lds, w, c0, split, splits, slot);
    }
}

// Joins the slots of a (row, head), D / 4 lanes each.  Bound by latency: the statistics of all slots come in one load (lane i: slot i), the accumulators eight slots at a time.
#define PA_MAX_SLOTS 32
#define PA_OWN_SLOTS 8  // of them, at most for the own keys where there is a prefix
template <int D>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(isst_prefix_attn a, PrefixPlan p) {
    constexpr int L4 = D / 4, E = PA_MAX_SLOTS / L4;
    const long pair = (long)blockIdx.x * (256 / L4) + threadIdx.x / L4, stride = (long)a.rows * a.heads;
    const int i = threadIdx.x % L4;
    if (pair >= stride) return;
    const int row = (int)(pair / a.heads), head = (int)(pair % a.heads);
    float m[E], w[E], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int s = i + e * L4;
        const float2 x = s < p.slots ? p.ml[s * stride + pair] : make_float2(-INFINITY, 0.f);
        m[e] = x.x; w[e] = x.y;
        M = fmaxf(M, x.x);
    }
    if (seq_of_row(a, row) < 0) return;
#pragma unroll
    for (int d = 1; d < L4; d <<= 1) M = fmaxf(M, __shfl_xor(M, d, WAVE));
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float l = w[e];
        w[e] = l == 0.f ? 0.f : m[e] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[e] - M);  // (no key: nothing; -inf with a sum: NaN scores only)
        L += l == 0.f ? 0.f : l * w[e];
    }
#pragma unroll
    for (int d = 1; d < L4; d <<= 1) L += __shfl_xor(L, d, WAVE);
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    const float* src = p.o + pair * D + 4 * i;
    for (int s0 = 0; s0 < p.slots; s0 += 8) {
        f32x4_t x[8];
        float ws[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int s = s0 + k;
            ws[k] = s < p.slots ? __shfl(E == 1 || s0 < L4 ? w[0] : w[E - 1], s % L4, L4) : 0.f;
            x[k] = ws[k] != 0.f ? *reinterpret_cast<const f32x4_t*>(src + s * stride * D) : (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) o += x[k] * ws[k];
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    const u32x2_t r = {pack_bf(o.x * inv, o.y * inv), pack_bf(o.z * inv, o.w * inv)};
    *reinterpret_cast<u32x2_t*>(a.out + row * a.out_row + head * a.out_head + 4 * i) = r;
}

// ---------------------------------------------------------------------------------------------------------------- host
// the launch's model, in microseconds: a tile of 128 columns in a full chip (128-wide heads), and what a unit costs beside its tiles (start, turning and storing its accumulators)
#define PA_TAU 1.0
#define PA_FIX 5.0
#define PA_MAX_UNITS (1L << 22)
static int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }
// most columns of a sequence that the launch is shaped for (of the hint, or the mean: a longer sequence walks on in its units)
static long own_columns(const isst_prefix_attn& a) {
    const int rows = a.row_starts ? (a.max_rows ? min(a.max_rows, a.rows) : ceil_div(a.rows, a.seqs)) : a.rows / a.seqs;
    return (long)(rows > 0 ? rows : 1) * (a.heads / a.kv_heads);
}
// Columns of a span: 16, or 32 where a sequence (or the batch, against the prefix) has 17 to 32: the keys are then read once (64 x 5 rows of 4 heads over 500 own keys: 39 us, as two spans of 16
// 44).  From 33 on the block role: at 40 columns 60 us against 58 as three spans, at 64 64 against 64, at 88 and more faster
static int span_nq(const isst_prefix_attn& a) {
    const long own = a.tail_cap > 0 ? own_columns(a) : 0, all = a.prefix_len > 0 ? (long)a.rows * (a.heads / a.kv_heads) : 0;
    return (own > 16 && own <= 32) || (all > 16 && all <= 32) ? 2 : 1;
}
static PrefixPlan plan(const isst_prefix_attn& a) {
    PrefixPlan p{};
    const int G = a.heads / a.kv_heads, nq = span_nq(a), width = 32 * PA_NW;
    p.magic = G > 1 ? (unsigned)(((1ull << 32) + G - 1) / G) : 0;
    const long cols = (long)a.rows * G;
    const double room = 256.0 * (8 / PA_NW);  // workgroups the chip runs at once
    double own_us = 0;                        // time of the own keys' units, summed
    if (a.tail_cap > 0) {
        const long oc = own_columns(a);
        p.own_block = oc > 32;
        p.own_tiles = ceil_div(oc, p.own_block ? width : 16 * nq);
        const long groups = (long)a.seqs * a.kv_heads, keys = p.own_block ? PA_TILE : 32 * PA_NW;
        while (p.own_tiles > 1 && groups * p.own_tiles > PA_MAX_UNITS) p.own_tiles = (p.own_tiles + 1) / 2;  // (a grid ends at 2^32 threads: the units walk on)
        p.own_splits = 1;
        const int most = a.prefix_len > 0 ? PA_OWN_SLOTS : PA_MAX_SLOTS;  // (one row over 100000 own keys: 8 spans 139 us, 32 83)
        while (p.own_splits < most && groups * p.own_tiles * p.own_splits * 2 <= room && p.own_splits * 2 <= ceil_div(a.tail_cap, (p.own_block ? 4 : 2) * keys)) p.own_splits *= 2;
        p.own_units = p.own_tiles * 8 * ceil_div(groups * p.own_splits, 8);
        own_us = (double)groups * p.own_tiles * (p.own_block ? a.tail_cap / 2 / (double)PA_TILE * PA_TAU : a.tail_cap / 2 * (4.0 * a.head_dim) / (20e3 * PA_NW / 8));
    }
    if (a.prefix_len > 0) {
        p.prefix_block = cols > 32;
        p.prefix_tiles = p.prefix_block ? ceil_div(cols, width) : 1;
        if (p.prefix_block) {
            // Key spans: the rounds of the chip that the units take (with the own keys' units filling what a last round leaves) + what their partial results cost
            const int tiles = ceil_div(a.prefix_len, PA_TILE), groups = a.kv_heads * p.prefix_tiles;
            double best = 1e30;
            for (int s = 1; s <= PA_MAX_SLOTS - PA_OWN_SLOTS && s <= tiles && (s == 1 || (long)groups * s <= PA_MAX_UNITS); ++s) {
                const int per = ceil_div(tiles, s);
                if (ceil_div(tiles, per) != s) continue;
                const double dur = per * PA_TAU * (a.head_dim / 128.0) + PA_FIX, units = (double)groups * s;
                const double even = (units * dur + own_us) / room, rounds = dur * ceil_div((long)units, (long)room);
                const double t = (even > rounds ? even : rounds) + s * (double)a.rows * a.heads * (8.0 * a.head_dim) / 3e6;
                if (t < best) { best = t; p.prefix_splits = s; }
            }
        } else {
            p.prefix_splits = ceil_div(a.prefix_len, 32 * PA_NW);
            if (p.prefix_splits > PA_MAX_SLOTS - PA_OWN_SLOTS) p.prefix_splits = PA_MAX_SLOTS - PA_OWN_SLOTS;
        }
        p.prefix_units = p.prefix_tiles * 8 * ceil_div((long)a.kv_heads * p.prefix_splits, 8);
    }
    p.slots = p.prefix_splits + p.own_splits;
    return p;
}
int64_t prefix_attention_workspace(const isst_prefix_attn& a) {
    return (int64_t)plan(a).slots * a.rows * a.heads * (a.head_dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
}
template <int D, int NQ>
static void launch_partial(const isst_prefix_attn& a, const PrefixPlan& p, hipStream_t s) {
    hipLaunchKernelGGL((prefix_attn_partial_kernel<D, PA_NW, NQ>), dim3((unsigned)(p.prefix_units + p.own_units)), dim3(PA_NW * 64), 0, s, a, p);
}
int launch_prefix_attention(const isst_prefix_attn& a, void* workspace, hipStream_t s) {
    PrefixPlan p = plan(a);
    const long pairs = (long)a.rows * a.heads;
    p.o = static_cast<float*>(workspace);
    p.ml = reinterpret_cast<float2*>(p.o + p.slots * pairs * a.head_dim);
    const int nq = span_nq(a);
    if (p.prefix_units + p.own_units > 0) {
        if (a.head_dim == 128) { if (nq == 1) launch_partial<128, 1>(a, p, s); else launch_partial<128, 2>(a, p, s); }
        else { if (nq == 1) launch_partial<64, 1>(a, p, s); else launch_partial<64, 2>(a, p, s); }
    }
    if (a.head_dim == 128) hipLaunchKernelGGL(prefix_attn_join_kernel<128>, dim3((unsigned)((pairs + 7) / 8)), dim3(256), 0, s, a, p);
    else hipLaunchKernelGGL(prefix_attn_join_kernel<64>, dim3((unsigned)((pairs + 15) / 16)), dim3(256), 0, s, a, p);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
