// A shared projection with a low-rank adapter per row (gfx950): out[m] = bf16(base[m] + scale_a up_a (down_a x[m])), a = the row's adapter.
// base = x W^T comes from the packed-weight GEMM as fp32 K slices (their sum is the base; it is never rounded on its own).
//
// Both kernels take tiles of 16 rows and walk the DISTINCT adapters of a tile: one matrix product per adapter for all 16 rows, of which every row keeps the one of its own adapter -- a
// selection, so that another adapter's inf or NaN cannot reach it.  No sorting and no plan: neighbouring rows of a stream share an adapter (one or two products a tile), and a decode
// step with an adapter per row reads each adapter once, as it has to.  Bound by the adapters' bytes and, below them, by latency.
// Measured next to their base product (us, down + base + up; K x N, rank, rows): 4096 x 6144, 16, 1 row 3.9 + 8.7 + 3.9; 64 rows with 64 adapters 5.1 + 18 + 7.0; 14336 x 4096, 64, 320 rows
// 12 + 48 + 14.3; 4096 x 4096, 32, 1408 rows 8.2 + 46 + 17.2.
#include "common.h"
#include "kernels.h"

#define LORA_ROWS 16
#define LORA_DOWN_WAVES 4
#define LORA_STEP_K (LORA_DOWN_WAVES * 64)  // k of a workgroup's step
typedef __attribute__((address_space(3))) void* lora_lds_ptr;
#define LORA_K_SLICE 1024  // k of a workgroup
#define LORA_FULL 1024     // workgroups up to which the adapters of a tile go to several
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

// t[slice][m][r] = the K slice's part of down[a][r] . x[m].  Units: row tile fastest, then z of Z, then K slice; adapter j of a tile belongs to z = j mod Z.
// A fragment read straight from memory is 64 pieces of 16 bytes to the L1 cache, a cycle each, and that was what bound this kernel: through LDS-DMA, eight rows of whole lines an instruction and a step
// ahead, 320 rows of 14336 x 64 16.5 -> 12.5 us, 1408 rows of 4096 x 32 10 -> 8.2.  K slices of 512 / 1024 / 2048 a workgroup: 320 rows 13 / 12.5 / 12.5, and the up kernel has the fewer slices to
// add (19 / 17.2 / 16.3); one row 4.1 / 4.0 / 4.7, 64 rows 5.2 / 5.2 / 6.2, 1408 rows 8.1 / 8.2 / 8.8
template <int RT>  // rank tiles of 16
__global__ __launch_bounds__(LORA_DOWN_WAVES * 64) void lora_down_kernel(LoraArgs g, int tiles, int Z, int units) {
    constexpr int TILE = LORA_ROWS * 128, BUF = (1 + RT) * TILE, LOADS = 2 * (1 + RT);  // bytes of 16 rows x 64 k; x and the rank tiles; LDS-DMA instructions a step
    __shared__ __attribute__((aligned(1024))) char lds[LORA_DOWN_WAVES * 2 * BUF];   // two steps a wave, then the waves' sums (ONE object: see prefix_attn.hip)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
    const int unit = xcd_unit(blockIdx.x, units);
    if (unit < 0) return;
    const int tile = unit % tiles, z = unit / tiles % Z, slice = unit / tiles / Z;
    const int m0 = tile * LORA_ROWS, k0 = slice * LORA_K_SLICE, steps = (min(LORA_K_SLICE, g.K - k0) + LORA_STEP_K - 1) / LORA_STEP_K;
    unsigned leaders;
    const int id = tile_ids(g, m0, leaders);
    unsigned mine = 0, done = 0;  // the first rows of this workgroup's adapters; all rows of them
    int j = 0;
    for (unsigned l = leaders; l; l &= l - 1, ++j)
        if (j % Z == z) {
            mine |= l & -l;
            done |= (unsigned)__ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctz(l))) & 0xffffu;
        }
    if (!done) return;  // (uniform over the workgroup)
    int id4[4];         // ids of the rows 4 fq + r that this lane's accumulators belong to
#pragma unroll
    for (int r = 0; r < 4; ++r) id4[r] = __shfl(id, 4 * fq + r, WAVE);

    // a step of a wave: 64 k of the 16 rows and of the adapter's rank rows, 8 rows of 128 bytes an instruction; the swizzle is in which chunk of its row a lane asks for
    char* const ring = lds + wave * (2 * BUF);
    const int dr = lane >> 3, dc = 8 * ((lane & 7) ^ dr);
    const bf16_t* xrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) xrow[i] = g.A + (long)min(m0 + 8 * i + dr, g.M - 1) * g.lda;
    auto ask = [&](int a, int step, char* buf) {
        const int k = min(k0 + step * LORA_STEP_K + wave * 64 + dc, g.K - 8);  // (past the end: something, unused)
        const bf16_t* w = g.down + (long)a * g.rank * g.K + k;
#pragma unroll
        for (int i = 0; i < 2; ++i) __builtin_amdgcn_global_load_lds((const void*)(xrow[i] + k), (lora_lds_ptr)(buf + 1024 * i), 16, 0, 0);
#pragma unroll
        for (int n = 0; n < RT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                __builtin_amdgcn_global_load_lds((const void*)(w + (long)min(16 * n + 8 * i + dr, g.rank - 1) * g.K), (lora_lds_ptr)(buf + (1 + n) * TILE + 1024 * i), 16, 0, 0);
    };
    f32x4_t t[RT], acc[RT];
#pragma unroll
    for (int n = 0; n < RT; ++n) t[n] = acc[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    unsigned ahead = mine;  // adapter and step that are asked for next
    int astep = 0, turn = 0;
    auto ask_next = [&](char* buf) {
        ask(__builtin_amdgcn_readlane(id, __builtin_ctz(ahead)), astep, buf);
        if (++astep == steps) { astep = 0; ahead &= ahead - 1; }
    };
    ask_next(ring);
    for (; mine; mine &= mine - 1) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(mine));
        for (int step = 0; step < steps; ++step, ++turn) {
            const char* buf = ring + (turn & 1) * BUF;
            if (ahead) {
                ask_next(ring + (~turn & 1) * BUF);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (k0 + step * LORA_STEP_K + wave * 64 + 32 * s >= g.K) break;
                const int off = fr * 128 + 16 * ((4 * s + fq) ^ (fr & 7));
                const bf16x8_t xf = __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(buf + off));
#pragma unroll
                for (int n = 0; n < RT; ++n)
                    acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4_t*>(buf + (1 + n) * TILE + off)), acc[n], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);  // (the fragments have been read before the step after next is asked for)
        }
#pragma unroll
        for (int n = 0; n < RT; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (id4[r] == a) t[n][r] = acc[n][r];
            acc[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }
    }
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);  // [waves][16 rows][16 RT]
#pragma unroll
    for (int n = 0; n < RT; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[(wave * LORA_ROWS + 4 * fq + r) * (RT * 16) + 16 * n + fr] = t[n][r];
    __syncthreads();
    for (int e = tid; e < LORA_ROWS * RT * 16; e += LORA_DOWN_WAVES * 64) {
        const int row = e / (RT * 16), r = e % (RT * 16);
        if (!(done >> row & 1) || r >= g.rank) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < LORA_DOWN_WAVES; ++w) sum += red[(w * LORA_ROWS + row) * (RT * 16) + r];
        g.t[((long)slice * g.M + m0 + row) * g.rank + r] = sum;
    }
}

// Units: row tile fastest, then column tile of 64 CG.  t enters the product as a pair of bf16 numbers (hi, lo: 2^-15 relative) side by side along the product's depth, both against the same entries
// of up.  CG = 1: the waves take an adapter each (few workgroups: decode steps; 64 rows with 64 adapters 6.9 us, with CG = 4 13.5); CG = 4: a column group each
// (t is summed once for 256 columns: 1408 rows 19 us, with CG = 1 26).  Bound by the base's fp32 slices: 46 MB at 1408 rows, 42 MB at 320
template <int RT, int CG>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs g, int tiles, int units) {
    constexpr int LD = RT * 16 + 8;  // (row padding: the rows of a fragment start in different banks)
    constexpr int UB = CG == 1 ? 0 : 64 * RT * 32, TH = 2 * LORA_ROWS * LD * 2, DL = LORA_ROWS * (64 * CG + 4) * 4;
    __shared__ __attribute__((aligned(1024))) char lds[4 * UB + TH + DL];  // a wave's 64 rows of an adapter; t; the adapters' sum (ONE object: see prefix_attn.hip)
    typedef bf16_t th_t[LORA_ROWS][LD];
    typedef float delta_t[64 * CG + 4];
    th_t* const th = reinterpret_cast<th_t*>(lds + 4 * UB);
    delta_t* const delta = reinterpret_cast<delta_t*>(lds + 4 * UB + TH);
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
    const int R8 = g.rank / 8, cg = CG == 1 ? 0 : wave;
    // CG = 4: an adapter's rows n0 + 64 cg .. + 63 lie in one piece and go through LDS, 1 KB of whole lines an instruction (fragments read from memory are 64 pieces of 16 bytes: 320 rows of rank
    // 64 82.5 -> 78.9 us in all); chunks of a row swizzled (where their number is a power of two) in which one a lane asks for.  CG = 1: fragments straight from memory (64 rows 30.0 us, through
    // LDS 31.3: one round trip less)
    char* const ubuf = lds + wave * UB;
    const int mask = R8 & (R8 - 1) ? 0 : (R8 - 1) & 7;
    const unsigned magic = (unsigned)((0x100000000ull + R8 - 1) / R8);
    auto ask = [&](int a) {
        const bf16_t* up = g.up + (long)a * g.N * g.rank;
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i)
            if (i < R8) {
                const int q = 64 * i + lane, row = R8 > 1 ? (int)__umulhi((unsigned)q, magic) : q, c = (q - row * R8) ^ (row & mask);
                __builtin_amdgcn_global_load_lds((const void*)(up + (long)min(n0 + 64 * cg + row, g.N - 1) * g.rank + 8 * c), (lora_lds_ptr)(ubuf + 1024 * i), 16, 0, 0);
            }
    };
    if (leaders) {
        if (CG > 1) ask(__builtin_amdgcn_readlane(id, __builtin_ctz(leaders)));
        const int slices = (g.K + LORA_K_SLICE - 1) / LORA_K_SLICE;
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
            // hi = the bf16 number below |v| and never v itself, so that lo has v's sign and is zero only where v is: an infinite entry of up times the pair is then up times v, and no v below
            // fp32's end rounds to infinity (v infinite: hi finite, lo infinite)
            f32x4_t hi, lo;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned bits = __float_as_uint(v[k]);
                hi[k] = __uint_as_float((bits - ((bits & 0x7fffffffu) != 0u)) & 0xffff0000u);
                lo[k] = v[k] - hi[k];
            }
            *reinterpret_cast<u32x2_t*>(&th[0][row][r]) = (u32x2_t){pack_bf(hi.x, hi.y), pack_bf(hi.z, hi.w)};
            *reinterpret_cast<u32x2_t*>(&th[1][row][r]) = (u32x2_t){pack_bf(lo.x, lo.y), pack_bf(lo.z, lo.w)};
        }
        __syncthreads();
        const int steps = (2 * R8 + 3) / 4;
        int j = 0;
        for (unsigned l = leaders; l; l &= l - 1, ++j) {
            if (CG == 1 && (j & 3) != wave) continue;
            const int a = __builtin_amdgcn_readlane(id, __builtin_ctz(l));
            f32x4_t acc[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            if constexpr (CG > 1) {
                if (j > 0) ask(a);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            const bf16_t* up = g.up + (long)a * g.N * g.rank;
            constexpr int U = CG > 1 || RT < 2 ? 1 : 2;  // steps whose fragments are in flight together
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
                        if constexpr (CG > 1) uf[u][c] = live ? *reinterpret_cast<const u32x4_t*>(ubuf + (16 * c + fr) * (2 * g.rank) + 16 * (r8 ^ (fr & mask))) : zero;
                        else uf[u][c] = live && n < g.N ? *reinterpret_cast<const u32x4_t*>(up + (long)n * g.rank + 8 * r8) : zero;
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
            __builtin_amdgcn_sched_barrier(0);  // (the fragments have been read before the next adapter is asked for)
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

static int k_slices(int K) { return (K + LORA_K_SLICE - 1) / LORA_K_SLICE; }
int64_t lora_t_floats(int M, int N, int K, int rank, int n_adapters) { return (int64_t)k_slices(K) * M * rank; }
template <int RT>
static void launch_down(const LoraArgs& g, hipStream_t s) {
    const int tiles = (g.M + LORA_ROWS - 1) / LORA_ROWS, ks = k_slices(g.K);
    int z = 1;  // adapters of a tile over several workgroups while the chip has room
    while (z < 16 && z * 2 <= g.M && z * 2 <= g.n_adapters && (long)tiles * ks * z * 2 <= LORA_FULL) z *= 2;
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
