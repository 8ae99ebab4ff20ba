// Verification of drafted tokens (gfx950): accept draft x_i while u_i q_i(x_i) < p_i(x_i), then draw from max(p_i - q_i, 0) or, with every draft accepted, from p_n.
// p, q = softmax of fp32 score rows.  Everything behind the scores is in 64 bits: the outcome of a comparison or of a draw must not depend on the order of a sum, and with
// 32-bit probabilities the borders of the inverse CDF move by ~1e-8 each -- over 128 k of them one draw in a thousand would land elsewhere.
#include "common.h"
#include "kernels.h"

#define VF_THREADS 256
struct VerifyStat { double sum; float max; int at; };
// sum over the workgroup in a fixed order (thread 0 .. 255 through LDS), in every thread
__device__ __forceinline__ double block_sum(double v, double* sh) {
    __syncthreads();
    sh[threadIdx.x] = v;
    __syncthreads();
    for (int s = VF_THREADS / 2; s > 0; s >>= 1) {
        if ((int)threadIdx.x < s) sh[threadIdx.x] += sh[threadIdx.x + s];
        __syncthreads();
    }
    return sh[0];
}

// per row: maximum, its first index, sum of exp(score - maximum); maximum = NaN for a row without a distribution
__global__ __launch_bounds__(VF_THREADS) void verify_stats_kernel(VerifyArgs g) {
    __shared__ double sh[VF_THREADS];
    __shared__ float smax[VF_THREADS];
    __shared__ int sidx[VF_THREADS], sbad[VF_THREADS];
    const int rows_t = g.max_drafts + 1, per = rows_t + (g.draft ? g.max_drafts : 0), tid = threadIdx.x;
    const int b = blockIdx.x / per, i = blockIdx.x % per;
    const float* x = i < rows_t ? g.target + b * g.target_stream + i * g.target_row : g.draft + b * g.draft_stream + (i - rows_t) * g.draft_row;
    float m = -INFINITY;
    int at = 0x7fffffff, bad = 0;
    for (int v = tid; v < g.vocab; v += VF_THREADS) {
        const float s = x[v];
        bad |= !(s < INFINITY);  // NaN or +inf
        if (s > m) { m = s; at = v; }
    }
    smax[tid] = m; sidx[tid] = at; sbad[tid] = bad;
    __syncthreads();
    for (int s = VF_THREADS / 2; s > 0; s >>= 1) {
        if (tid < s) {
            if (smax[tid + s] > smax[tid] || (smax[tid + s] == smax[tid] && sidx[tid + s] < sidx[tid])) { smax[tid] = smax[tid + s]; sidx[tid] = sidx[tid + s]; }
            sbad[tid] |= sbad[tid + s];
        }
        __syncthreads();
    }
    m = smax[0];
    const bool ok = !sbad[0] && m > -INFINITY;
    double sum = 0.0;
    if (ok)
        for (int v = tid; v < g.vocab; v += VF_THREADS) sum += exp((double)x[v] - (double)m);
    sum = block_sum(sum, sh);
    if (tid == 0) {
        VerifyStat st;
        st.sum = sum; st.max = ok ? m : NAN; st.at = sidx[0];
        static_cast<VerifyStat*>(g.workspace)[blockIdx.x] = st;
    }
}

// per stream: the acceptances, then the draw
__global__ __launch_bounds__(VF_THREADS) void verify_draw_kernel(VerifyArgs g) {
    __shared__ double sh[VF_THREADS];
    __shared__ int s_at, s_last;
    const int b = blockIdx.x, tid = threadIdx.x, K = g.max_drafts, rows_t = K + 1, per = rows_t + (g.draft ? K : 0);
    const VerifyStat *st = static_cast<const VerifyStat*>(g.workspace) + (long)b * per, *sq = st + rows_t;
    const int* x = g.drafts + (long)b * K;
    const int n = g.n_drafts ? g.n_drafts[b] : K;
    bool bad = n < 0 || n > K;
    int i = 0;
    for (; !bad && i < n; ++i) {
        if (st[i].max != st[i].max || x[i] < 0 || x[i] >= g.vocab || (g.draft && sq[i].max != sq[i].max)) { bad = true; break; }
        if (!g.uniforms) {
            if (x[i] != st[i].at) break;
            continue;
        }
        const double u = g.uniforms[(long)b * (K + 1) + i];
        if (!(u >= 0.0 && u < 1.0)) { bad = true; break; }
        const double p = exp((double)g.target[b * g.target_stream + i * g.target_row + x[i]] - (double)st[i].max) / st[i].sum;
        const double q = g.draft ? exp((double)g.draft[b * g.draft_stream + i * g.draft_row + x[i]] - (double)sq[i].max) / sq[i].sum : 1.0;
        if (!(u * q < p)) break;
    }
    if (!bad && st[i].max != st[i].max) bad = true;
    const double u = g.uniforms ? g.uniforms[(long)b * (K + 1) + K] : 0.0;
    if (!(u >= 0.0 && u < 1.0)) bad = true;
    int pick = -1;
    if (!bad && !g.uniforms) pick = st[i].at;
    if (!bad && g.uniforms) {
        const float* t = g.target + b * g.target_stream + i * g.target_row;
        const float* dq = g.draft ? g.draft + b * g.draft_stream + i * g.draft_row : nullptr;
        const int chunk = (g.vocab + VF_THREADS - 1) / VF_THREADS, lo = min(tid * chunk, g.vocab), hi = min(lo + chunk, g.vocab);
        for (int pass = i < n ? 0 : 1; pass < 2; ++pass) {  // 0: what the draft left over, 1: the row itself
            auto weight = [&](int v) {
                const double p = exp((double)t[v] - (double)st[i].max) / st[i].sum;
                if (pass == 1) return p;
                if (!dq) return v == x[i] ? 0.0 : p;
                return fmax(p - exp((double)dq[v] - (double)sq[i].max) / sq[i].sum, 0.0);
            };
            double mine = 0.0;
            for (int v = lo; v < hi; ++v) mine += weight(v);
            __syncthreads();
            sh[tid] = mine;
            if (tid == 0) { s_at = 0x7fffffff; s_last = -1; }
            __syncthreads();
            double before = 0.0, total = 0.0;
            for (int k = 0; k < VF_THREADS; ++k) {
                if (k < tid) before += sh[k];
                total += sh[k];
            }
            if (!(total > 0.0)) continue;
            const double goal = u * total;
            double cum = before;
            int last = -1;
            if (mine > 0.0 && before + mine > goal)
                for (int v = lo; v < hi; ++v) {
                    const double w = weight(v);
                    if (!(w > 0.0)) continue;
                    cum += w;
                    if (cum > goal) { atomicMin(&s_at, v); break; }
                }
            if (mine > 0.0)
                for (int v = lo; v < hi; ++v)
                    if (weight(v) > 0.0) last = v;
            atomicMax(&s_last, last);
            __syncthreads();
            pick = s_at < g.vocab ? s_at : s_last;
            break;
        }
    }
    if (tid == 0) {
        if (pick < 0) bad = true;
        for (int k = 0; k <= K; ++k) g.tokens[(long)b * (K + 1) + k] = bad ? -1 : k < i ? x[k] : k == i ? pick : -1;
        g.counts[b] = bad ? -1 : i + 1;
    }
}

int64_t verify_workspace(int streams, int max_drafts, int) { return (int64_t)streams * (2 * max_drafts + 1) * (int64_t)sizeof(VerifyStat); }
int launch_verify(const VerifyArgs& g, hipStream_t s) {
    const int per = g.max_drafts + 1 + (g.draft ? g.max_drafts : 0);
    hipLaunchKernelGGL(verify_stats_kernel, dim3((unsigned)(g.streams * per)), dim3(VF_THREADS), 0, s, g);
    hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)g.streams), dim3(VF_THREADS), 0, s, g);
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
