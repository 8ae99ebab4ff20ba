// A shared projection with a low-rank adapter per row (gfx950): out[m] = bf16(base[m] + scale_a up_a (down_a x[m])), a = the row's adapter.
// base = x W^T comes from the packed-weight GEMM as fp32 K slices (their sum is the base; it is never rounded on its own).
//
// Both kernels take tiles of 16 rows and walk the DISTINCT adapters of a tile: one matrix product per adapter for all 16 rows, of which every row keeps the one of its own adapter -- a
// selection, so that another adapter's inf or NaN cannot reach it.  No sorting and no plan: neighbouring rows of a stream share an adapter (one or two products a tile), and a decode
// step with an adapter per row reads each adapter once, as it has to.  Bound by the adapters' bytes and, below them, by latency.
// Measured next to their base product (us, down + base + up; K x N, rank, rows): 4096 x 6144, 16, 1 row 3.9 + 8.9 + 3.9; 64 rows with 64 adapters 5.3 + 18 + 7.0; 14336 x 4096, 64, 320 rows
// 16.5 + 49 + 17; 4096 x 4096, 32, 1408 rows 10 + 51 + 19.
#include "common.h"
#include "kernels.h"

#define LORA_ROWS 16
#define LORA_DOWN_WAVES 4
#define LORA_STEPS 4                                     // 32-deep product steps of a wave
#define LORA_DOWN_K (LORA_DOWN_WAVES * LORA_STEPS * 32)  // K slice of a workgroup
#define LORA_WIDE 256  // workgroups of 256 columns a row tile from which these are taken instead of 64

// the tile's adapters: id of row lane & 15 in every lane (-1: none), and which rows are the first of their adapter
__device__ __forceinline__ int tile_ids(const LoraArgs& g, int m0, unsigned& leaders) {
    const int lane = threadIdx.x & 63, m = m0 + (lane & 15);
    int id = m < g.M ? g.row_adapter[m] : -1;
    if (id < 0 || id >= g.n_adapters) id = -1;
    leaders = 0;
#pragma unroll
    for (int i = 0; i < LORA_ROWS; ++i) {
        const int a = __builtin_amdgcn_readlane(id, i);
        const unsigned same = (unsigned)__ballot(id == a) & 0xffffu;
        if (a >= 0 && __builtin_ctz(same) == i) leaders |= 1u << i;
    }
    return id;
}

// Workgroup i runs on XCD i % 8, each with an L2 of its own: gives every XCD a contiguous eighth of `total` units, so that units that read the same adapter share an L2.  < 0: none left
__device__ __forceinline__ int xcd_unit(int i, int total) {
    const int per = (total + 7) / 8, u = (i & 7) * per + (i >> 3);
    return (i >> 3) < per && u < total ? u : -1;
}

// t[slice][m][r] = the K slice's part of down[a][r] . x[m].  Slices of 512 = four waves x four product steps (256 or 1024 a workgroup: 1408 rows 10 -> 11 or 12.5 us, 320 rows 16.5 -> 15 or 20,
// and the up kernel has twice or half the slices to add: 17 -> 20 or 17; 32-row tiles: the same).  Units: row tile fastest, then z of Z, then K slice; adapter j of a tile belongs to z = j mod Z
template <int RT>  // rank tiles of 16
__global__ __launch_bounds__(LORA_DOWN_WAVES * 64) void lora_down_kernel(LoraArgs g, int tiles, int Z, int units) {
    __shared__ float red[LORA_DOWN_WAVES][LORA_ROWS][RT * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int unit = xcd_unit(blockIdx.x, units);
    if (unit < 0) return;
    const int tile = unit % tiles, z = unit / tiles % Z, slice = unit / tiles / Z;
    const int m0 = tile * LORA_ROWS, k0 = slice * LORA_DOWN_K + wave * (LORA_STEPS * 32) + 8 * fq;
    unsigned leaders;
    const int id = tile_ids(g, m0, leaders);
    u32x4_t xf[LORA_STEPS];
    const u32x4_t zero = {0u, 0u, 0u, 0u};
    const bf16_t* x = g.A + (long)min(m0 + fr, g.M - 1) * g.lda;
#pragma unroll
    for (int s = 0; s < LORA_STEPS; ++s) xf[s] = k0 + 32 * s < g.K ? *reinterpret_cast<const u32x4_t*>(x + k0 + 32 * s) : zero;
    int id4[4];  // ids of the rows 4 fq + r that this lane's accumulators belong to
#pragma unroll
    for (int r = 0; r < 4; ++r) id4[r] = __shfl(id, 4 * fq + r, WAVE);
    f32x4_t t[RT];
#pragma unroll
    for (int n = 0; n < RT; ++n) t[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    unsigned done = 0;  // rows whose adapter is this workgroup's
    int j = 0;
    for (unsigned l = leaders; l; l &= l - 1, ++j) {
        if (j % Z != z) continue;
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(l));
        done |= (unsigned)__ballot(id == a) & 0xffffu;
        const bf16_t* w = g.down + (long)a * g.rank * g.K;
        u32x4_t wf[RT][LORA_STEPS];  // (all of them in flight before the first product: one round trip per adapter)
#pragma unroll
        for (int n = 0; n < RT; ++n)
#pragma unroll
            for (int s = 0; s < LORA_STEPS; ++s)
                wf[n][s] = k0 + 32 * s < g.K ? *reinterpret_cast<const u32x4_t*>(w + (long)min(16 * n + fr, g.rank - 1) * g.K + k0 + 32 * s) : zero;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < RT; ++n) {
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < LORA_STEPS; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, xf[s]), __builtin_bit_cast(bf16x8_t, wf[n][s]), acc, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (id4[r] == a) t[n][r] = acc[r];
        }
    }
    if (!done) return;  // (uniform over the workgroup)
#pragma unroll
    for (int n = 0; n < RT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[wave][4 * fq + r][16 * n + fr] = t[n][r];
    __syncthreads();
    for (int e = tid; e < LORA_ROWS * RT * 16; e += LORA_DOWN_WAVES * 64) {
        const int row = e / (RT * 16), r = e % (RT * 16);
        if (!(done >> row & 1) || r >= g.rank) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < LORA_DOWN_WAVES; ++w) s += red[w][row][r];
        g.t[((long)slice * g.M + m0 + row) * g.rank + r] = s;
    }
}

// Units: row tile fastest, then column tile of 64 CG.  t enters the product as a pair of bf16 numbers (hi, lo: 2^-16 relative) side by side along the product's depth, both against the same entries
// of up.  CG = 1: the waves take an adapter each (few workgroups: decode steps; 64 rows with 64 adapters 6.9 us, with CG = 4 13.5); CG = 4: a column group each
// (t is summed once for 256 columns: 1408 rows 19 us, with CG = 1 26).  Bound by the base's fp32 slices: 46 MB at 1408 rows, 42 MB at 320
template <int RT, int CG>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs g, int tiles, int units) {
    constexpr int LD = RT * 16 + 8;  // (row padding: the rows of a fragment start in different banks)
    __shared__ __attribute__((aligned(16))) bf16_t th[2][LORA_ROWS][LD];
    __shared__ __attribute__((aligned(16))) float delta[LORA_ROWS][64 * CG + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int unit = xcd_unit(blockIdx.x, units);
    if (unit < 0) return;
    const int m0 = unit % tiles * LORA_ROWS, n0 = unit / tiles * 64 * CG;
    // this thread's outputs, four per column group: the first two slices of their base are asked for first, everything else hides behind them
    const int orow = tid >> 4, ocol = (tid & 15) * 4, om = min(m0 + orow, g.M - 1);
    f32x4_t base[2][CG];
    const float* bp = g.base + (long)om * g.ld_base;
    const long slab = (long)g.M * g.ld_base;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < CG; ++c)
            base[s][c] = s < g.slabs ? *reinterpret_cast<const f32x4_t*>(bp + s * slab + min(n0 + 64 * c + ocol, (int)g.ld_base - 4)) : (f32x4_t){0.f, 0.f, 0.f, 0.f};

    unsigned leaders;
    const int id = tile_ids(g, m0, leaders);
    if (leaders) {
        const int slices = (g.K + LORA_DOWN_K - 1) / LORA_DOWN_K;
        const int r4s = g.rank / 4;
        for (int e = tid; e < LORA_ROWS * r4s; e += 256) {  // four entries of a row, eight slices in flight
            const int row = e / r4s, r = 4 * (e - row * r4s), m = m0 + row, a = m < g.M ? g.row_adapter[m] : -1;
            f32x4_t v = {0.f, 0.f, 0.f, 0.f};
            if (a >= 0 && a < g.n_adapters) {
                const float* tp = g.t + (long)m * g.rank + r;
                const long ts = (long)g.M * g.rank;
                const float scale = g.scales[a];
                for (int s0 = 0; s0 < slices; s0 += 8) {
                    f32x4_t x[8];
#pragma unroll
                    for (int s = 0; s < 8; ++s) x[s] = s0 + s < slices ? *reinterpret_cast<const f32x4_t*>(tp + (s0 + s) * ts) : (f32x4_t){0.f, 0.f, 0.f, 0.f};
                    v += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
                }
                v *= scale;
            }
            f32x4_t lo;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float hi = bfr(v[k]);
                lo[k] = __builtin_isfinite(hi) ? v[k] - hi : 0.f;
            }
            *reinterpret_cast<u32x2_t*>(&th[0][row][r]) = (u32x2_t){pack_bf(v.x, v.y), pack_bf(v.z, v.w)};
            *reinterpret_cast<u32x2_t*>(&th[1][row][r]) = (u32x2_t){pack_bf(lo.x, lo.y), pack_bf(lo.z, lo.w)};
        }
        __syncthreads();
        const int R8 = g.rank / 8, steps = (2 * R8 + 3) / 4, cg = CG == 1 ? 0 : wave;
        int j = 0;
        for (unsigned l = leaders; l; l &= l - 1, ++j) {
            if (CG == 1 && (j & 3) != wave) continue;
            const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(l));
            f32x4_t acc[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            const bf16_t* up = g.up + (long)a * g.N * g.rank;
            constexpr int U = RT < 2 ? 1 : 2;  // steps whose fragments are in flight together
            for (int s0 = 0; s0 < steps; s0 += U) {
                u32x4_t uf[U][4], tf[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int ch = 4 * (s0 + u) + fq, part = ch >= R8, r8 = part ? ch - R8 : ch;
                    const bool live = ch < 2 * R8;
                    const u32x4_t zero = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int n = n0 + 64 * cg + 16 * c + fr;
                        uf[u][c] = live && n < g.N ? *reinterpret_cast<const u32x4_t*>(up + (long)n * g.rank + 8 * r8) : zero;
                    }
                    tf[u] = live ? *reinterpret_cast<const u32x4_t*>(&th[part][fr][8 * r8]) : zero;
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, uf[u][c]), __builtin_bit_cast(bf16x8_t, tf[u]), acc[c], 0, 0, 0);
            }
            if (id == a)
#pragma unroll
                for (int c = 0; c < 4; ++c) *reinterpret_cast<f32x4_t*>(&delta[fr][64 * cg + 16 * c + 4 * fq]) = acc[c];
        }
        __syncthreads();
    }
    for (int s0 = 2; s0 < g.slabs; s0 += 2) {
        f32x4_t x[2][CG];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int c = 0; c < CG; ++c)
                x[s][c] = s0 + s < g.slabs ? *reinterpret_cast<const f32x4_t*>(bp + (s0 + s) * slab + min(n0 + 64 * c + ocol, (int)g.ld_base - 4)) : (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CG; ++c) base[0][c] += x[0][c] + x[1][c];
    }
    if (m0 + orow >= g.M) return;
    const int a = g.row_adapter[m0 + orow];
#pragma unroll
    for (int c = 0; c < CG; ++c) {
        const int n = n0 + 64 * c + ocol;
        if (n >= g.N) break;
        f32x4_t y = base[0][c] + base[1][c];
        if (a >= 0 && a < g.n_adapters) y += *reinterpret_cast<const f32x4_t*>(&delta[orow][64 * c + ocol]);
        bf16_t* out = g.out + (m0 + orow) * g.ldo + n;
        const u32x2_t v = {pack_bf(y.x, y.y), pack_bf(y.z, y.w)};
        if (n + 4 <= g.N && !(reinterpret_cast<uintptr_t>(out) & 7)) *reinterpret_cast<u32x2_t*>(out) = v;
        else
            for (int e = 0; e < 4; ++e)
                if (n + e < g.N) out[e] = (bf16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
}

static int k_slices(int K) { return (K + LORA_DOWN_K - 1) / LORA_DOWN_K; }
int64_t lora_t_floats(int M, int N, int K, int rank, int n_adapters) { return (int64_t)k_slices(K) * M * rank; }
template <int RT>
static void launch_down(const LoraArgs& g, hipStream_t s) {
    const int tiles = (g.M + LORA_ROWS - 1) / LORA_ROWS, ks = k_slices(g.K);
    int z = 1;  // adapters of a tile over several workgroups while the chip has room
    while (z < 16 && z * 2 <= g.M && z * 2 <= g.n_adapters && (long)tiles * ks * z * 2 <= 512) z *= 2;
    const int units = tiles * ks * z;
    hipLaunchKernelGGL(lora_down_kernel<RT>, dim3((units + 7) / 8 * 8), dim3(LORA_DOWN_WAVES * 64), 0, s, g, tiles, z, units);
}
int launch_lora_down(const LoraArgs& g, hipStream_t s) {
    if (g.rank <= 16) launch_down<1>(g, s);
    else if (g.rank <= 32) launch_down<2>(g, s);
    else if (g.rank <= 64) launch_down<4>(g, s);
    else launch_down<8>(g, s);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
template <int CG>
static void launch_up(const LoraArgs& g, hipStream_t s) {
    const int tiles = (g.M + LORA_ROWS - 1) / LORA_ROWS, units = tiles * ((g.N + 64 * CG - 1) / (64 * CG));
    const dim3 grid((units + 7) / 8 * 8);
    if (g.rank <= 16) hipLaunchKernelGGL((lora_up_kernel<1, CG>), grid, dim3(256), 0, s, g, tiles, units);
    else if (g.rank <= 32) hipLaunchKernelGGL((lora_up_kernel<2, CG>), grid, dim3(256), 0, s, g, tiles, units);
    else if (g.rank <= 64) hipLaunchKernelGGL((lora_up_kernel<4, CG>), grid, dim3(256), 0, s, g, tiles, units);
    else hipLaunchKernelGGL((lora_up_kernel<8, CG>), grid, dim3(256), 0, s, g, tiles, units);
}
int launch_lora_up(const LoraArgs& g, hipStream_t s) {
    const long groups = (long)((g.M + LORA_ROWS - 1) / LORA_ROWS) * ((g.N + 63) / 64);
    if (groups >= 4 * LORA_WIDE) launch_up<4>(g, s);
    else launch_up<1>(g, s);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
