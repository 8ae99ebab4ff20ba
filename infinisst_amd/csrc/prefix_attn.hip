// Attention of a batch whose sequences share one long prefix in front of keys of their own (gfx950).
//
// Row t of the n rows of sequence b sees the P prefix keys and its own keys j < len_b - n + t + 1:
//     o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)   over both sets, m = the running maximum.
// One launch computes partial (O, m, l) triples, a second one joins them.  A workgroup of the first launch takes one of two roles:
//   block: 32 NW columns ((row, head) pairs of one key head, over ALL sequences) against a span of the prefix.  Every K / V tile of 64 keys goes through LDS once for all columns.
//   span:  16 NQ columns of ONE sequence against its own keys (or of the whole batch against the prefix where it has no more columns than that); the waves split the keys.
// Scores are computed transposed, S^T = K Q^T, so that a lane holds one column: statistics and rescaling are per lane, and the exponentials are already in the layout the value product
// O^T = V^T P^T wants its B operand in (the order of the keys inside a 16- or 32-key step is free as long as V^T is read in the same order: two transposed LDS reads).
#include "../../include/infinisst_hip.h"
#include "common.h"
#include "kernels.h"

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

#define PA_TILE 64               // keys of a block tile
// Keys and values are read through buffer descriptors that start at a tile's first row: a lane's offset is either its row's (rows lie up to 2^25 bytes apart, 63 of them stay inside the
// descriptor) or PA_OOB, for which the load returns zeros -- also with the scalar offset of the row group added.
#define PA_EXTENT 0x7fffffffu
#define PA_OOB 0x80000000u

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
    int col_tiles, prefix_splits, split_tiles;  // block form: column tiles, key spans of split_tiles tiles.  col_tiles = 0: the prefix runs in span form
    int own_tiles, own_splits;                  // span form of the own keys: column tiles of a sequence (a longer one walks on), key splits
    int prefix_units, own_units, slots;
    float* o;                                   // [slots][rows * heads][D] fp32, unnormalised
    float2* ml;                                 // [slots][rows * heads]: maximum (in units of log2), sum
};

// XOR swizzle of the 16-byte chunks of a K / V tile row: 16 rows read at one chunk (K fragments) and 4 rows x 4 chunks (transposed V reads) both cover all 64 banks once
template <int D>
__device__ __forceinline__ int tile_off(int row, int ch) {
    if constexpr (D == 128) return 256 * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3)));
    return 128 * row + 16 * (ch ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)));
}
__device__ __forceinline__ u32x2_t read_tr(const char* p) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)p));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t key_rsrc(const bf16_t* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(p), 0, PA_EXTENT, 0x00020000);
}

// ---------------------------------------------------------------------------------------------------------------- block role
template <int D, int NW>
__device__ __forceinline__ void block_role(const isst_prefix_attn& a, const PrefixPlan& p, int unit, char* lds) {
    constexpr int ROWB = 2 * D, CH = D / 8, LOADS = PA_TILE * CH / (NW * 64), RSTEP = NW * 64 / CH, QS = D / 16, DT = D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, half = lane >> 5;
    const int split = unit % p.prefix_splits, ct = (unit / p.prefix_splits) % p.col_tiles, kvh = unit / p.prefix_splits / p.col_tiles;
    const int G = a.heads / a.kv_heads, cols = a.rows * G;
    const int tile0 = split * p.split_tiles, tiles = min(p.split_tiles, (a.prefix_len + PA_TILE - 1) / PA_TILE - tile0);
    const int col = (ct * NW + wave) * 32 + c32;
    const bool live = col < cols, wave_live = (ct * NW + wave) * 32 < cols;
    const int row = live ? col / G : 0, head = kvh * G + (live ? col % G : 0);

    u32x4_t qf[QS];
#pragma unroll
    for (int s = 0; s < QS; ++s) qf[s] = live ? *reinterpret_cast<const u32x4_t*>(a.q + row * a.q_row + head * a.q_head + 16 * s + 8 * half) : (u32x4_t){0u, 0u, 0u, 0u};

    const bf16_t *kb = a.k_prefix + kvh * a.kp_head, *vb = a.v_prefix + kvh * a.vp_head;
    const int lr = tid / CH, lc = tid % CH, kstep = (int)a.kp_key * 2, vstep = (int)a.vp_key * 2;
    const unsigned koff = lr * kstep + lc * 16, voff = lr * vstep + lc * 16;
    u32x4_t ks[LOADS], vs[LOADS];
    auto fetch = [&](int t) {
        const int j0 = (tile0 + t) * PA_TILE, rows = min(PA_TILE, a.prefix_len - j0);
        const __amdgpu_buffer_rsrc_t kr = key_rsrc(kb + j0 * a.kp_key), vr = key_rsrc(vb + j0 * a.vp_key);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            ks[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, lr < rows - i * RSTEP ? koff : PA_OOB, i * RSTEP * kstep, 0);
            vs[i] = __builtin_amdgcn_raw_buffer_load_b128(vr, lr < rows - i * RSTEP ? voff : PA_OOB, i * RSTEP * vstep, 0);
        }
    };
    auto put = [&](int buf) {
        char* base = lds + buf * (2 * PA_TILE * ROWB);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            *reinterpret_cast<u32x4_t*>(base + tile_off<D>(lr + i * RSTEP, lc)) = ks[i];
            *reinterpret_cast<u32x4_t*>(base + PA_TILE * ROWB + tile_off<D>(lr + i * RSTEP, lc)) = vs[i];
        }
    };
    f32x16_t o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float c2 = a.scale * 1.44269504088896340736f;  // exp(scale s - ..) = exp2(c2 s - ..)

    fetch(0);
    put(0);
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
        if (t + 1 < tiles) fetch(t + 1);
        const char* kt = lds + (t & 1) * (2 * PA_TILE * ROWB);
        const char* vt = kt + PA_TILE * ROWB;
        if (wave_live) {
            f32x16_t sc[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[u][r] = 0.f;
#pragma unroll
                for (int s = 0; s < QS; ++s) {
                    const u32x4_t kf = *reinterpret_cast<const u32x4_t*>(kt + tile_off<D>(32 * u + c32, 2 * s + half));
                    sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kf), __builtin_bit_cast(bf16x8_t, qf[s]), sc[u], 0, 0, 0);
                }
            }
            const int rows = a.prefix_len - (tile0 + t) * PA_TILE;
            if (rows < PA_TILE) {  // the prefix ends inside this tile
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (32 * u + (r & 3) + 8 * (r >> 2) + 4 * half >= rows) sc[u][r] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[u][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE)) * c2;
            if (__any(mx > m)) {
                const float m2 = fmaxf(m, mx), keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m2);
                l *= keep;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= keep;
                m = m2;
            }
            const float neg = m == -INFINITY ? 0.f : -m;
            u32x4_t pf[4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float e[16];
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][r], c2, neg));
                    l += e[r];
                }
#pragma unroll
                for (int kb2 = 0; kb2 < 2; ++kb2)
                    pf[2 * u + kb2] = (u32x4_t){pack_bf(e[8 * kb2], e[8 * kb2 + 1]), pack_bf(e[8 * kb2 + 2], e[8 * kb2 + 3]), pack_bf(e[8 * kb2 + 4], e[8 * kb2 + 5]), pack_bf(e[8 * kb2 + 6], e[8 * kb2 + 7])};
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // 16 keys: slots j < 4 of half h = keys 16 k + 4 h + j, j >= 4 = keys 16 k + 8 + 4 h + (j - 4)
                    const int r = 16 * k + 4 * half + ((lane >> 2) & 3);
                    const u32x2_t v1 = read_tr(vt + tile_off<D>(r, ch) + 8 * (lane & 1)), v2 = read_tr(vt + tile_off<D>(r + 8, ch) + 8 * (lane & 1));
                    const u32x4_t vf = {v1.x, v1.y, v2.x, v2.y};
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf), __builtin_bit_cast(bf16x8_t, pf[k]), o[d], 0, 0, 0);
                }
            }
        }
        if (t + 1 < tiles) put((t + 1) & 1);
        __syncthreads();
    }
    if (!live) return;
    l += __shfl_xor(l, 32, WAVE);
    const long at = (long)split * a.rows * a.heads + (long)row * a.heads + head;
    if (half == 0) p.ml[at] = make_float2(m, l);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
            *reinterpret_cast<f32x4_t*>(p.o + at * D + 32 * d + 8 * r4 + 4 * half) = (f32x4_t){o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
}

// ---------------------------------------------------------------------------------------------------------------- span role
// keys 0 .. see(last column) of (kb, vb) for columns [c0, c0 + 16 NQ) of `ncols` (column c = row first + c / G, head kvh G + c % G); column c sees keys j < limit0 + c / G (limit0 < 0: all `keys`)
template <int D, int NW, int NQ>
__device__ __forceinline__ void span_role(const isst_prefix_attn& a, const PrefixPlan& p, char* lds, int kvh, int first, int c0, int ncols, const bf16_t* kb, long kstride, const bf16_t* vb,
                                          long vstride, int keys, bool causal, int limit0, int split, int splits, int slot) {
    constexpr int ROWB = 2 * D, CH = D / 8, VL = 32 * CH / 64, VR = 64 / CH, QS = D / 32, NT = D / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int G = a.heads / a.kv_heads;
    int limit[NQ];
    u32x4_t qf[NQ][QS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int c = c0 + 16 * n + fr;
        const bool live = c < ncols;
        const int row = first + (live ? c / G : 0), head = kvh * G + (live ? c % G : 0);
        limit[n] = causal && live ? min(max(limit0 + c / G, 0), keys) : keys;
#pragma unroll
        for (int s = 0; s < QS; ++s) qf[n][s] = live ? *reinterpret_cast<const u32x4_t*>(a.q + row * a.q_row + head * a.q_head + 32 * s + 8 * fq) : (u32x4_t){0u, 0u, 0u, 0u};
    }
    const int last = min(c0 + 16 * NQ, ncols) - 1;
    const int see_least = causal ? min(max(limit0 + c0 / G, 0), keys) : keys, see_most = causal ? min(max(limit0 + last / G, 0), keys) : keys;

    f32x4_t o[NQ][NT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -INFINITY; l[n] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[n][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    const float c2 = a.scale * 1.44269504088896340736f;
    char* vl = lds + wave * (32 * ROWB);
    u32x4_t kf[2][QS], vr[VL];
    const int kstep = (int)kstride * 2, vstep = (int)vstride * 2;
    const unsigned koff = fr * kstep + 16 * fq, voff = lane / CH * vstep + 16 * (lane % CH);
    auto fetch_k = [&](int j0) {
        const __amdgpu_buffer_rsrc_t r = key_rsrc(kb + j0 * kstride);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const unsigned off = fr < see_most - j0 - 16 * t ? koff : PA_OOB;
#pragma unroll
            for (int s = 0; s < QS; ++s) kf[t][s] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 16 * t * kstep + 64 * s, 0);
        }
    };
    auto fetch_v = [&](int j0) {
        const __amdgpu_buffer_rsrc_t r = key_rsrc(vb + j0 * vstride);
#pragma unroll
        for (int i = 0; i < VL; ++i) vr[i] = __builtin_amdgcn_raw_buffer_load_b128(r, lane / CH < see_most - j0 - i * VR ? voff : PA_OOB, i * VR * vstep, 0);
    };
    const int step = 32 * NW * splits;
    int j0 = 32 * (split * NW + wave);
    if (j0 < see_most) { fetch_v(j0); fetch_k(j0); }
    for (; j0 < see_most; j0 += step) {
#pragma unroll
        for (int i = 0; i < VL; ++i) *reinterpret_cast<u32x4_t*>(vl + tile_off<D>(i * VR + lane / CH, lane % CH)) = vr[i];
        const bool more = j0 + step < see_most;
        if (more) fetch_v(j0 + step);
        __builtin_amdgcn_sched_barrier(0);
        f32x4_t sc[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                sc[n][t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < QS; ++s)
                    sc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[t][s]), __builtin_bit_cast(bf16x8_t, qf[n][s]), sc[n][t], 0, 0, 0);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (more) fetch_k(j0 + step);
        __builtin_amdgcn_sched_barrier(0);
        const bool edge = j0 + 32 > see_least;  // some column does not see some key of this step
        u32x4_t pf[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            if (edge) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (j0 + 16 * t + 4 * fq + r >= limit[n]) sc[n][t][r] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[n][t][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, WAVE));
            mx = fmaxf(mx, __shfl_xor(mx, 32, WAVE)) * c2;
            const float m2 = fmaxf(m[n], mx), keep = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - m2), neg = m2 == -INFINITY ? 0.f : -m2;
            l[n] *= keep;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[n][t][r] *= keep;
            m[n] = m2;
            float e[8];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    e[4 * t + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][t][r], c2, neg));
                    l[n] += e[4 * t + r];
                }
            pf[n] = (u32x4_t){pack_bf(e[0], e[1]), pack_bf(e[2], e[3]), pack_bf(e[4], e[5]), pack_bf(e[6], e[7])};
        }
        if (edge) {
            bool ill = false;  // inf or NaN among the values of a step that not every column sees whole
#pragma unroll 1
            for (int i = 0; i < VL; ++i) {
                const u32x4_t v = *reinterpret_cast<const u32x4_t*>(vl + 1024 * i + 16 * lane);
#pragma unroll
                for (int w = 0; w < 4; ++w) ill |= (v[w] & 0x7f80u) == 0x7f80u || (v[w] & 0x7f800000u) == 0x7f800000u;
            }
            if (__any(ill)) {
                // 0 x inf must not reach a column that does not see the key: the keys that every column sees go through the matrix product below, the others (they see_least ..
                // see_most of this step) are added here where they are seen and their rows cleared
                int vb = fq;
                asm volatile("" : "+v"(vb));  // (keeps this block's addresses out of the loop's preheader: they would take the registers of the ordinary path)
#pragma unroll 1
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int key = 16 * (k >> 2) + 4 * q + (k & 3);
                        if (j0 + key < see_least) continue;
                        float pk[NQ];
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            const uint32_t w = (uint32_t)__shfl((int)pf[n][k >> 1], 16 * q + fr, WAVE);
                            pk[n] = (k & 1) ? hi_bf(w) : lo_bf(w);
                        }
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            const u32x2_t v = *reinterpret_cast<const u32x2_t*>(vl + tile_off<D>(key, 2 * t + (vb >> 1)) + 8 * (vb & 1));
#pragma unroll
                            for (int n = 0; n < NQ; ++n)
                                if (j0 + key < limit[n]) {
                                    o[n][t][0] += pk[n] * lo_bf(v.x); o[n][t][1] += pk[n] * hi_bf(v.x);
                                    o[n][t][2] += pk[n] * lo_bf(v.y); o[n][t][3] += pk[n] * hi_bf(v.y);
                                }
                        }
                    }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < VL; ++i)
                    if (j0 + i * VR + lane / CH >= see_least) *reinterpret_cast<u32x4_t*>(vl + tile_off<D>(i * VR + lane / CH, lane % CH) + (vb - fq)) = (u32x4_t){0u, 0u, 0u, 0u};
                __builtin_amdgcn_wave_barrier();
            }
        }
        const int vrow = 4 * fq + ((lane >> 2) & 3), vch = (lane & 3) >> 1, vb8 = 8 * (lane & 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const u32x2_t v1 = read_tr(vl + tile_off<D>(vrow, 2 * t + vch) + vb8), v2 = read_tr(vl + tile_off<D>(16 + vrow, 2 * t + vch) + vb8);
            const u32x4_t vf = {v1.x, v1.y, v2.x, v2.y};
            if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (four fragments ahead at most: more of them spill)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
                o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vf), __builtin_bit_cast(bf16x8_t, pf[n]), o[n][t], 0, 0, 0);
        }
    }
    // ---- join the waves: statistics first, then the weighted accumulators of 16 columns at a time ----
    int jt = tid;
    asm volatile("" : "+v"(jt));  // (keeps this part's addresses out of the registers of the loop above)
    const int jc = jt & 15, jq = (jt & 63) >> 4;
    __shared__ float2 wml[NW][16 * NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor(l[n], 16, WAVE);
        l[n] += __shfl_xor(l[n], 32, WAVE);
        if (jq == 0) wml[wave][16 * n + jc] = make_float2(m[n], l[n]);
    }
    __syncthreads();  // (also: every wave is done with its value tile, which the accumulators overlay)
    float* red = reinterpret_cast<float*>(lds);  // [NW][16 columns][D]
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, wml[w][16 * n + jc].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float2 x = wml[w][16 * n + jc];
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
            const int cc = c0 + 16 * n + c;
            if (cc < ncols) {
                const long at = (long)slot * a.rows * a.heads + (long)(first + cc / G) * a.heads + kvh * G + cc % G;
                *reinterpret_cast<f32x4_t*>(p.o + at * D + 4 * d4) = s;
            }
        }
        if (wave == 0 && jq == 0 && c0 + 16 * n + jc < ncols) {
            const int cc = c0 + 16 * n + jc;
            p.ml[(long)slot * a.rows * a.heads + (long)(first + cc / G) * a.heads + kvh * G + cc % G] = make_float2(M, L);
        }
        __syncthreads();
    }
}

template <int D, int NW, int NQ>
__global__ __launch_bounds__(NW * 64, 2) void prefix_attn_partial_kernel(isst_prefix_attn a, PrefixPlan p) {
    constexpr int BLOCK_LDS = 4 * PA_TILE * 2 * D, SPAN_LDS = NW * 16 * D * 4;
    __shared__ __attribute__((aligned(16))) char lds[BLOCK_LDS > SPAN_LDS ? BLOCK_LDS : SPAN_LDS];
    int unit = blockIdx.x;
    const bool prefix = unit < p.prefix_units;
    if (prefix && p.col_tiles) {
        block_role<D, NW>(a, p, unit, lds);
        return;
    }
    // span role: of the own keys of a sequence, or of the prefix for a batch of no more than one column tile
    if (!prefix) unit -= p.prefix_units;
    const int splits = prefix ? p.prefix_splits : p.own_splits, tiles = prefix ? 1 : p.own_tiles;
    const int split = unit % splits, ct = unit / splits % tiles, kvh = unit / splits / tiles % a.kv_heads, b = unit / splits / tiles / a.kv_heads, G = a.heads / a.kv_heads;
    int first = 0, n = a.rows, keys = a.prefix_len, limit0 = a.prefix_len;
    if (!prefix) {
        seq_rows(a, b, first, n);
        first = __builtin_amdgcn_readfirstlane(first);  // (uniform already; a value the compiler keeps in a vector register would make every key load a loop over lanes)
        n = __builtin_amdgcn_readfirstlane(n);
        keys = __builtin_amdgcn_readfirstlane(a.tail_lens[b]);
        keys = min(max(keys, 0), a.tail_cap);
        limit0 = keys - n + 1;
    }
    const bf16_t* kb = prefix ? a.k_prefix + kvh * a.kp_head : a.k_tail + b * a.kt_seq + kvh * a.kt_head;
    const bf16_t* vb = prefix ? a.v_prefix + kvh * a.vp_head : a.v_tail + b * a.vt_seq + kvh * a.vt_head;
    for (int c0 = ct * 16 * NQ; c0 < n * G; c0 += tiles * 16 * NQ)
        span_role<D, NW, NQ>(a, p, lds, kvh, first, c0, n * G, kb, prefix ? a.kp_key : a.kt_key, vb, prefix ? a.vp_key : a.vt_key, keys, !prefix, limit0, split, splits,
                             prefix ? split : p.prefix_splits + split);
}

// joins the slots of a (row, head): D / 4 lanes each
template <int D>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(isst_prefix_attn a, PrefixPlan p) {
    constexpr int L4 = D / 4;
    const long pair = (long)blockIdx.x * (256 / L4) + threadIdx.x / L4;
    const int d4 = threadIdx.x % L4;
    if (pair >= (long)a.rows * a.heads) return;
    const int row = (int)(pair / a.heads), head = (int)(pair % a.heads);
    if (seq_of_row(a, row) < 0) return;
    const long stride = (long)a.rows * a.heads;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < p.slots; ++s) M = fmaxf(M, p.ml[s * stride + pair].x);
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.slots; ++s) {
        const float2 x = p.ml[s * stride + pair];
        if (x.y == 0.f) continue;  // no key
        const float w = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.x - M);  // (-inf with a sum: NaN scores only)
        L += x.y * w;
        o += *reinterpret_cast<const f32x4_t*>(p.o + (s * stride + pair) * D + 4 * d4) * w;
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    const u32x2_t r = {pack_bf(o.x * inv, o.y * inv), pack_bf(o.z * inv, o.w * inv)};
    *reinterpret_cast<u32x2_t*>(a.out + row * a.out_row + head * a.out_head + 4 * d4) = r;
}

// ---------------------------------------------------------------------------------------------------------------- host
#define PA_NW 8
static int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }
static int span_nq(const isst_prefix_attn& a) {
    const int G = a.heads / a.kv_heads, rows = a.row_starts ? (a.max_rows ? a.max_rows : ceil_div(a.rows, a.seqs)) : a.rows / a.seqs;
    return (long)rows * G > 16 ? 2 : 1;
}
static PrefixPlan plan(const isst_prefix_attn& a) {
    PrefixPlan p{};
    const int G = a.heads / a.kv_heads, nq = span_nq(a);
    const long cols = (long)a.rows * G;
    if (a.prefix_len > 0) {
        if (cols <= 16 * nq) {
            p.prefix_splits = ceil_div(a.prefix_len, 32 * PA_NW);
            if (p.prefix_splits > 32) p.prefix_splits = 32;
            p.prefix_units = a.kv_heads * p.prefix_splits;
        } else {
            p.col_tiles = ceil_div(cols, 32 * PA_NW);
            const int tiles = ceil_div(a.prefix_len, PA_TILE), base = a.kv_heads * p.col_tiles;
            int splits = base >= 256 ? 1 : 256 / base;
            if (splits > tiles) splits = tiles;
            p.split_tiles = ceil_div(tiles, splits);
            p.prefix_splits = ceil_div(tiles, p.split_tiles);
            p.prefix_units = base * p.prefix_splits;
        }
    }
    if (a.tail_cap > 0) {
        const int rows = a.row_starts ? (a.max_rows ? a.max_rows : ceil_div(a.rows, a.seqs)) : a.rows / a.seqs;
        p.own_tiles = ceil_div((long)(rows > 0 ? rows : 1) * G, 16 * nq);
        const long units = (long)a.seqs * a.kv_heads * p.own_tiles;
        p.own_splits = 1;
        while (p.own_splits < 16 && units * p.own_splits * 2 <= 256 && p.own_splits * 2 <= ceil_div(a.tail_cap, 32 * PA_NW)) p.own_splits *= 2;
        p.own_units = (int)(units * p.own_splits);
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
