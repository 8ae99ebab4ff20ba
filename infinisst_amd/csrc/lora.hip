// A shared projection with a low-rank adapter per row (gfx950): out[m] = bf16(base[m] + scale_a * up_a (down_a x[m])), a = the row's adapter.
// base = x W^T comes from the packed-weight GEMM as fp32 K slices (their sum is the base; it is never rounded on its own).
#include "common.h"
#include "kernels.h"

// t[m][r] = down[a][r] . x[m]: one wave per (m, r)
__global__ __launch_bounds__(64) void lora_down_kernel(LoraArgs g) {
    const int m = blockIdx.x / g.rank, r = blockIdx.x % g.rank, a = g.row_adapter[m];
    if (a < 0 || a >= g.n_adapters) return;
    const bf16_t *x = g.A + m * g.lda, *w = g.down + ((long)a * g.rank + r) * g.K;
    float s = 0.f;
    for (int k = threadIdx.x; k < g.K; k += 64) s += bf2f(x[k]) * bf2f(w[k]);
    s = wave_sum(s);
    if (threadIdx.x == 0) g.t[(long)m * g.rank + r] = s;
}
// one thread per output
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs g) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= g.N) return;
    for (int m = blockIdx.y; m < g.M; m += gridDim.y) {
        float s = 0.f;
        for (int k = 0; k < g.slabs; ++k) s += g.base[((long)k * g.M + m) * g.ld_base + n];
        const int a = g.row_adapter[m];
        if (a >= 0 && a < g.n_adapters) {
            const bf16_t* u = g.up + ((long)a * g.N + n) * g.rank;
            float d = 0.f;
            for (int r = 0; r < g.rank; ++r) d += g.t[(long)m * g.rank + r] * bf2f(u[r]);
            s += g.scales[a] * d;
        }
        g.out[m * g.ldo + n] = f2bf(s);
    }
}

int64_t lora_t_floats(int M, int, int, int rank, int) { return (int64_t)M * rank; }
int launch_lora_down(const LoraArgs& g, hipStream_t s) {
    hipLaunchKernelGGL(lora_down_kernel, dim3((unsigned)((long)g.M * g.rank)), dim3(64), 0, s, g);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
int launch_lora_up(const LoraArgs& g, hipStream_t s) {
    hipLaunchKernelGGL(lora_up_kernel, dim3((g.N + 255) / 256, g.M < 32768 ? g.M : 32768), dim3(256), 0, s, g);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
