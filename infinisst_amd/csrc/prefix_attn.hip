// Attention of a batch whose sequences share one long prefix in front of keys of their own (gfx950).
//
// Row t of the n rows of sequence b sees the P prefix keys and its own keys j < len_b - n + t + 1:
//     o = sum_j exp(scale q.k_j - m) v_j / sum_j exp(scale q.k_j - m)   over both sets, m = the running maximum.
#include "../../include/infinisst_hip.h"
#include "common.h"
#include "kernels.h"

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

// One wave per (row, head): a lane per key for the scores, a lane per two (one) dims for the values.
template <int D>
__global__ __launch_bounds__(64) void prefix_attn_row_kernel(isst_prefix_attn a) {
    const int row = blockIdx.x / a.heads, h = blockIdx.x % a.heads, kvh = h / (a.heads / a.kv_heads), lane = threadIdx.x;
    const int b = seq_of_row(a, row);
    if (b < 0) return;
    int first, n;
    seq_rows(a, b, first, n);
    __shared__ float qs[D];
    const bf16_t* q = a.q + row * a.q_row + h * a.q_head;
    for (int d = lane; d < D; d += 64) qs[d] = bf2f(q[d]) * a.scale;
    __syncthreads();
    constexpr int E = D / 64;
    float m = -INFINITY, l = 0.f, o[E] = {};
    auto walk = [&](const bf16_t* k, int64_t k_key, const bf16_t* v, int64_t v_key, int keys) {
        for (int j0 = 0; j0 < keys; j0 += 64) {
            float s = -INFINITY;
            if (j0 + lane < keys) {
                const bf16_t* kr = k + (j0 + lane) * k_key;
                s = 0.f;
                for (int d = 0; d < D; d += 8) {
                    float f[8];
                    unpack8(*reinterpret_cast<const u32x4_t*>(kr + d), f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s += f[e] * qs[d + e];
                }
            }
            const float m2 = fmaxf(m, wave_max(s)), safe = m2 == -INFINITY ? 0.f : m2;
            const float keep = expf(m - safe), p = expf(s - safe);
            l = l * keep + wave_sum(p);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= keep;
            const int cnt = min(64, keys - j0);
            for (int j = 0; j < cnt; ++j) {
                const float pj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), j));
                const bf16_t* vr = v + (j0 + j) * v_key + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += pj * bf2f(vr[e]);
            }
            m = m2;
        }
    };
    walk(a.k_prefix + kvh * a.kp_head, a.kp_key, a.v_prefix + kvh * a.vp_head, a.vp_key, a.prefix_len);
    const int len = min(max(a.tail_lens[b], 0), a.tail_cap);
    walk(a.k_tail + b * a.kt_seq + kvh * a.kt_head, a.kt_key, a.v_tail + b * a.vt_seq + kvh * a.vt_head, a.vt_key, len - n + (row - first) + 1);
    bf16_t* out = a.out + row * a.out_row + h * a.out_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = f2bf(l != 0.f ? o[e] / l : 0.f);
}

int64_t prefix_attention_workspace(const isst_prefix_attn&) { return 0; }
int launch_prefix_attention(const isst_prefix_attn& a, void*, hipStream_t s) {
    const dim3 grid((unsigned)((long)a.rows * a.heads));
    if (a.head_dim == 128) hipLaunchKernelGGL(prefix_attn_row_kernel<128>, grid, dim3(64), 0, s, a);
    else hipLaunchKernelGGL(prefix_attn_row_kernel<64>, grid, dim3(64), 0, s, a);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
