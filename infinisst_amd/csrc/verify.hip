// Verification of drafted tokens (gfx950): accept draft x_i while u_i q_i(x_i) < p_i(x_i), then draw from max(p_i - q_i, 0) or, with every draft accepted, from p_n.
// p, q = softmax of fp32 score rows.  Everything behind the scores is in 64 bits: the outcome of a comparison or of a draw must not depend on the order of a sum, and with
// 32-bit probabilities the borders of the inverse CDF move by ~1e-8 each -- over 128 k of them one draw in a thousand would land elsewhere.
//
// Launch 1 reads every score row once, a workgroup per slice of VF_SLICE entries (maximum, its first index, sum of exponentials); its floor is that read, and the 64-bit exponential (~20
// instructions) is short enough to hide behind it.  Launch 2 runs only where drafts bring scores: it sums what a refused draft leaves over, slice by slice.  Launch 3 takes one workgroup
// per stream: decide, find the slice that the draw falls into from the slice sums, walk that slice.
#include "common.h"
#include "kernels.h"

#define VF_THREADS 256
#define VF_PER 16                          // entries of a lane
#define VF_SLICE (VF_THREADS * VF_PER)
#define VF_ROWS 32                         // drafts that are decided at a time

struct VerifyStat { double sum; float max; int at; };  // of a slice: sum of exp(score - max), max (NaN: a NaN or +inf among the scores), the maximum's first index

typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));  // (rows start anywhere)

// exp(d) for d <= 0: 2^k exp(r) with |r| <= ln 2 / 2 and the Taylor series up to r^11 / 11!, whose remainder is below 7e-15 relative.  NaN (-inf less -inf) and anything under -800: 0
__device__ __forceinline__ double exp_le0(double d) {
    d = fmax(d, -800.0);
    const double k = rint(d * 1.4426950408889634074);
    const double r = fma(-k, 0x1.abc9e3b39803fp-56, fma(-k, 0x1.62e42fefa39efp-1, d));  // ln 2 and what its rounding left
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0); p = fma(p, r, 1.0 / 362880.0); p = fma(p, r, 1.0 / 40320.0); p = fma(p, r, 1.0 / 5040.0); p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0); p = fma(p, r, 1.0 / 24.0); p = fma(p, r, 1.0 / 6.0); p = fma(p, r, 0.5); p = fma(p, r, 1.0); p = fma(p, r, 1.0);
    return ldexp(p, (int)k);
}
__device__ __forceinline__ double shfl_d(double v, int lane) {
    const unsigned long long u = __double_as_longlong(v);
    return __longlong_as_double(((unsigned long long)(unsigned)__shfl((int)(u >> 32), lane, WAVE) << 32) | (unsigned)__shfl((int)u, lane, WAVE));
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += shfl_d(v, (threadIdx.x & 63) ^ m);
    return v;
}
// sum over this lane and the lanes before it
__device__ __forceinline__ double wave_scan_d(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const double o = shfl_d(v, (threadIdx.x & 63) - m);
        if ((int)(threadIdx.x & 63) >= m) v += o;
    }
    return v;
}
__device__ __forceinline__ int slices(int vocab) { return (vocab + VF_SLICE - 1) / VF_SLICE; }
__device__ __forceinline__ int rows_of(const VerifyArgs& g) { return g.max_drafts + 1 + (g.draft ? g.max_drafts : 0); }
__device__ __forceinline__ const VerifyStat* stats_of(const VerifyArgs& g, int b, int row) {
    return static_cast<const VerifyStat*>(g.workspace) + ((long)b * rows_of(g) + row) * slices(g.vocab);
}
__device__ __forceinline__ double* left_of(const VerifyArgs& g, int b) {  // launch 2's slice sums
    return reinterpret_cast<double*>(static_cast<VerifyStat*>(g.workspace) + (long)g.streams * rows_of(g) * slices(g.vocab)) + (long)b * slices(g.vocab);
}
__device__ __forceinline__ const float* target_row(const VerifyArgs& g, int b, int i) { return g.target + b * g.target_stream + i * g.target_row; }
__device__ __forceinline__ const float* draft_row(const VerifyArgs& g, int b, int i) { return g.draft + b * g.draft_stream + i * g.draft_row; }

// grid (slices, score rows)
__global__ __launch_bounds__(VF_THREADS) void verify_stats_kernel(VerifyArgs g) {
    __shared__ VerifyStat part[VF_THREADS / 64];
    const int tid = threadIdx.x, wave = tid >> 6, rows_t = g.max_drafts + 1, per = rows_of(g);
    const int b = blockIdx.y / per, i = blockIdx.y % per, lo = blockIdx.x * VF_SLICE;
    const float* x = i < rows_t ? target_row(g, b, i) : draft_row(g, b, i - rows_t);
    float s[VF_PER];
    int bad = 0;
    // a lane's entries: four at lo + 4 tid, VF_SLICE / 4 further on, ..
#pragma unroll
    for (int q = 0; q < VF_PER / 4; ++q) {
        const int v = lo + (q * VF_THREADS + tid) * 4;
        if (v + 4 <= g.vocab) {
            const f32x4u_t f = *reinterpret_cast<const f32x4u_t*>(x + v);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * q + e] = f[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * q + e] = v + e < g.vocab ? x[v + e] : -INFINITY;
        }
    }
    float m = -INFINITY;
    int at = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < VF_PER; ++k) {
        bad |= !(s[k] < INFINITY);  // NaN or +inf
        if (s[k] > m) { m = s[k]; at = lo + ((k >> 2) * VF_THREADS + tid) * 4 + (k & 3); }
    }
    wave_argmax_all(m, at);
    double sum = 0.0;
    if (g.uniforms) {
#pragma unroll
        for (int k = 0; k < VF_PER; ++k) sum += exp_le0((double)s[k] - (double)m);
        sum = wave_sum_d(sum);
    }
    bad = __any(bad);
    if ((tid & 63) == 0) part[wave] = {sum, bad ? NAN : m, at};
    __syncthreads();
    if (tid == 0) {
        VerifyStat t = part[0];
        for (int w = 1; w < VF_THREADS / 64; ++w) {
            const VerifyStat o = part[w];
            if (!(t.max == t.max) || !(o.max == o.max)) { t.max = NAN; continue; }
            const float M = fmaxf(t.max, o.max);
            t.sum = t.sum * exp_le0((double)t.max - (double)M) + o.sum * exp_le0((double)o.max - (double)M);
            if (o.max > t.max) t.at = o.at;  // (equal: the lower index is the earlier one -- below)
            else if (o.max == t.max) t.at = min(t.at, o.at);
            t.max = M;
        }
        static_cast<VerifyStat*>(g.workspace)[(long)blockIdx.y * gridDim.x + blockIdx.x] = t;
    }
}

// one row's statistics from its slices, by one wave, in every lane; max = NaN: no distribution
__device__ __forceinline__ VerifyStat merge_row(const VerifyArgs& g, int b, int row) {
    const VerifyStat* st = stats_of(g, b, row);
    const int S = slices(g.vocab), lane = threadIdx.x & 63;
    VerifyStat t = {0.0, -INFINITY, 0x7fffffff};
    bool bad = false;
    for (int s = lane; s < S; s += 64) {
        const VerifyStat o = st[s];
        bad |= !(o.max == o.max);
        const float M = fmaxf(t.max, o.max);
        t.sum = t.sum * exp_le0((double)t.max - (double)M) + o.sum * exp_le0((double)o.max - (double)M);
        if (o.max > t.max) t.at = o.at;  // (slices come in index order: on equality the earlier one stays)
        t.max = M;
    }
    float M = t.max;
    int at = t.at;
    wave_argmax_all(M, at);
    t.sum = wave_sum_d(t.sum * exp_le0((double)t.max - (double)M));
    t.max = __any(bad) || M == -INFINITY ? NAN : M;
    t.at = at;
    return t;
}

struct Decision {
    int accepted, n;  // accepted < 0: no answer
    VerifyStat p, q;  // of the row that decides (q: of the refused draft's scores)
};
// by the whole workgroup, the same in every thread
__device__ __forceinline__ Decision decide(const VerifyArgs& g, int b) {
    __shared__ VerifyStat sp[VF_ROWS + 1], sq[VF_ROWS];
    __shared__ int s_stop, s_bad;
    const int K = g.max_drafts, tid = threadIdx.x, wave = tid >> 6;
    const int* x = g.drafts + (long)b * K;
    Decision d;
    d.n = g.n_drafts ? g.n_drafts[b] : K;
    d.accepted = -1;
    if (d.n < 0 || d.n > K) return d;
    for (int i0 = 0;; i0 += VF_ROWS) {
        const int cnt = min(VF_ROWS, d.n - i0);  // drafts of this turn; the row behind the last one is looked at as well
        for (int k = wave; k < 2 * cnt + 1; k += VF_THREADS / 64) {
            if (k <= cnt) {
                const VerifyStat t = merge_row(g, b, i0 + k);
                if ((tid & 63) == 0) sp[k] = t;
            } else if (g.draft) {
                const VerifyStat t = merge_row(g, b, K + 1 + i0 + k - cnt - 1);
                if ((tid & 63) == 0) sq[k - cnt - 1] = t;
            }
        }
        if (tid == 0) s_stop = cnt;
        __syncthreads();
        if (wave == 0) {  // a lane per draft
            bool ok = true, bad = false;
            if (tid < cnt) {
                const VerifyStat p = sp[tid];
                const int i = i0 + tid, xi = x[i];
                if (p.max != p.max || xi < 0 || xi >= g.vocab) bad = true;
                else if (!g.uniforms) ok = xi == p.at;
                else {
                    const double u = g.uniforms[(long)b * (K + 1) + i];
                    double q = 1.0;
                    if (!(u >= 0.0 && u < 1.0)) bad = true;
                    if (g.draft) {
                        if (sq[tid].max != sq[tid].max) bad = true;
                        else q = exp_le0((double)draft_row(g, b, i)[xi] - (double)sq[tid].max) / sq[tid].sum;
                    }
                    if (!bad) ok = u * q < exp_le0((double)target_row(g, b, i)[xi] - (double)p.max) / p.sum;
                }
            }
            const unsigned long long stops = __ballot(bad || !ok), bads = __ballot(bad);
            const int first = stops ? __builtin_ctzll(stops) : cnt;
            if (tid == 0) {
                s_stop = first;
                s_bad = stops ? (int)(bads >> first & 1) : (i0 + cnt == d.n && sp[cnt].max != sp[cnt].max);
            }
        }
        __syncthreads();
        const int stop = s_stop;
        if (s_bad) return d;
        if (stop < cnt || i0 + cnt == d.n) {
            d.accepted = i0 + stop;
            d.p = sp[stop];
            if (g.draft && stop < cnt) d.q = sq[stop];
            return d;
        }
        __syncthreads();
    }
}

// what is drawn from: kind 0 = what scores leave over, 1 = the row without the draft, 2 = the row
__device__ __forceinline__ double weight(int kind, const Decision& d, float t, float q, bool is_draft, double inv_p, double inv_q) {
    const double p = exp_le0((double)t - (double)d.p.max) * inv_p;
    if (kind == 2) return p;
    if (kind == 1) return is_draft ? 0.0 : p;
    return fmax(p - exp_le0((double)q - (double)d.q.max) * inv_q, 0.0);
}
// the lane's entries lo + VF_PER tid .. of the slice
__device__ __forceinline__ void weights(const VerifyArgs& g, int b, const Decision& d, int kind, int lo, double (&w)[VF_PER]) {
    const int i = d.accepted, v0 = lo + VF_PER * threadIdx.x, xi = kind == 1 ? g.drafts[(long)b * g.max_drafts + i] : -1;
    const float *t = target_row(g, b, i), *q = kind == 0 ? draft_row(g, b, i) : t;
    const double inv_p = 1.0 / d.p.sum, inv_q = kind == 0 ? 1.0 / d.q.sum : 0.0;
    float ts[VF_PER], qs[VF_PER];
#pragma unroll
    for (int k = 0; k < VF_PER; k += 4) {
        if (v0 + k + 4 <= g.vocab) {
            const f32x4u_t f = *reinterpret_cast<const f32x4u_t*>(t + v0 + k), h = *reinterpret_cast<const f32x4u_t*>(q + v0 + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) { ts[k + e] = f[e]; qs[k + e] = h[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ts[k + e] = v0 + k + e < g.vocab ? t[v0 + k + e] : -INFINITY;
                qs[k + e] = v0 + k + e < g.vocab ? q[v0 + k + e] : -INFINITY;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < VF_PER; ++k) w[k] = weight(kind, d, ts[k], qs[k], v0 + k == xi, inv_p, inv_q);
}
// inclusive sum over the workgroup's threads in thread order, and the total
__device__ __forceinline__ double block_scan(double v, double& total) {
    __shared__ double wsum[VF_THREADS / 64];
    const int wave = threadIdx.x >> 6;
    v = wave_scan_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) wsum[wave] = v;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < VF_THREADS / 64; ++w) {
        if (w < wave) before += wsum[w];
        total += wsum[w];
    }
    return before + v;
}
__device__ __forceinline__ double slice_sum(const VerifyArgs& g, int b, const Decision& d, int kind, int lo) {
    double w[VF_PER], mine = 0.0, total;
    weights(g, b, d, kind, lo, w);
#pragma unroll
    for (int k = 0; k < VF_PER; ++k) mine += w[k];
    block_scan(mine, total);
    return total;
}

// grid (slices, streams): what a refused draft with scores leaves over
__global__ __launch_bounds__(VF_THREADS) void verify_left_kernel(VerifyArgs g) {
    const Decision d = decide(g, blockIdx.y);
    if (d.accepted < 0 || d.accepted == d.n) return;
    const double s = slice_sum(g, blockIdx.y, d, 0, blockIdx.x * VF_SLICE);
    if (threadIdx.x == 0) left_of(g, blockIdx.y)[blockIdx.x] = s;
}

// one workgroup per stream
__global__ __launch_bounds__(VF_THREADS) void verify_draw_kernel(VerifyArgs g) {
    __shared__ int s_slice, s_live, s_at, s_last;
    __shared__ double s_before, s_total;
    const int b = blockIdx.x, tid = threadIdx.x, K = g.max_drafts, S = slices(g.vocab);
    const Decision d = decide(g, b);
    int pick = -1;
    bool bad = d.accepted < 0;
    if (!bad && !g.uniforms) pick = d.p.at;
    if (!bad && g.uniforms) {
        const double u = g.uniforms[(long)b * (K + 1) + K];
        bad = !(u >= 0.0 && u < 1.0);
        const VerifyStat* st = stats_of(g, b, d.accepted);
        for (int kind = bad ? 3 : d.accepted == d.n ? 2 : g.draft ? 0 : 1; kind < 3; kind = 2) {
            const int xs = kind == 1 ? g.drafts[(long)b * K + d.accepted] / VF_SLICE : -1;  // (the slice that the draft is taken out of is summed anew)
            const double without = kind == 1 ? slice_sum(g, b, d, 1, xs * VF_SLICE) : 0.0;
            auto of_slice = [&](int s) {
                return kind == 0 ? left_of(g, b)[s] : s == xs ? without : st[s].sum * exp_le0((double)st[s].max - (double)d.p.max) / d.p.sum;
            };
            if (tid < 64) {  // total, then the slice whose running sum first exceeds u total (none, by rounding: the last one that holds anything)
                double total = 0.0;
                for (int s0 = 0; s0 < S; s0 += 64) total += wave_sum_d(s0 + tid < S ? of_slice(s0 + tid) : 0.0);
                int slice = -1, live = -1;
                double before = 0.0, cum = 0.0;
                for (int s0 = 0; s0 < S && slice < 0; s0 += 64) {
                    const double v = s0 + tid < S ? of_slice(s0 + tid) : 0.0, c = cum + wave_scan_d(v);
                    const unsigned long long hit = __ballot(v > 0.0 && c > u * total), any = __ballot(v > 0.0);
                    const int at = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : -1;
                    if (at >= 0) { live = s0 + at; before = shfl_d(c - v, at); }
                    if (hit) slice = live;
                    cum = shfl_d(c, 63);
                }
                if (tid == 0) { s_slice = slice; s_live = live; s_before = before; s_total = total; s_at = 0x7fffffff; s_last = -1; }
            }
            __syncthreads();
            const double total = s_total, goal = s_slice < 0 ? INFINITY : u * total;
            const int slice = s_live;
            if (!(total > 0.0) || slice < 0) {  // nothing left over: the row itself
                __syncthreads();
                if (kind == 2) break;
                continue;
            }
            double w[VF_PER], mine = 0.0, all;
            weights(g, b, d, kind, slice * VF_SLICE, w);
#pragma unroll
            for (int k = 0; k < VF_PER; ++k) mine += w[k];
            double cum = s_before + (block_scan(mine, all) - mine);
            int at = 0x7fffffff, last = -1;
#pragma unroll
            for (int k = 0; k < VF_PER; ++k) {
                if (!(w[k] > 0.0)) continue;
                cum += w[k];
                last = slice * VF_SLICE + VF_PER * tid + k;
                if (cum > goal && at == 0x7fffffff) at = last;
            }
            if (at != 0x7fffffff) atomicMin(&s_at, at);
            if (last >= 0) atomicMax(&s_last, last);
            __syncthreads();
            pick = s_at != 0x7fffffff ? s_at : s_last;
            break;
        }
    }
    bad |= pick < 0;
    for (int k = tid; k <= K; k += VF_THREADS) g.tokens[(long)b * (K + 1) + k] = bad ? -1 : k < d.accepted ? g.drafts[(long)b * K + k] : k == d.accepted ? pick : -1;
    if (tid == 0) g.counts[b] = bad ? -1 : d.accepted + 1;
}

static int64_t n_slices(int vocab) { return ((int64_t)vocab + VF_SLICE - 1) / VF_SLICE; }
int64_t verify_workspace(int streams, int max_drafts, int vocab) {
    return streams * n_slices(vocab) * ((2 * (int64_t)max_drafts + 1) * (int64_t)sizeof(VerifyStat) + (int64_t)sizeof(double));
}
int launch_verify(const VerifyArgs& g, hipStream_t s) {
    const int64_t S = n_slices(g.vocab);
    const int per = g.max_drafts + 1 + (g.draft ? g.max_drafts : 0);
    // (the grid's second dimension ends at 65535: more streams go in several turns, each with the workspace of its own streams)
    const int turn = 65535 / per;
    for (int b0 = 0; b0 < g.streams; b0 += turn) {
        VerifyArgs t = g;
        t.streams = g.streams - b0 < turn ? g.streams - b0 : turn;
        t.target += b0 * g.target_stream;
        if (t.draft) t.draft += b0 * g.draft_stream;
        t.drafts += (int64_t)b0 * g.max_drafts;
        if (t.n_drafts) t.n_drafts += b0;
        if (t.uniforms) t.uniforms += (int64_t)b0 * (g.max_drafts + 1);
        t.tokens += (int64_t)b0 * (g.max_drafts + 1);
        t.counts += b0;
        t.workspace = static_cast<char*>(g.workspace) + verify_workspace(b0, g.max_drafts, g.vocab);
        hipLaunchKernelGGL(verify_stats_kernel, dim3((unsigned)S, (unsigned)(t.streams * per)), dim3(VF_THREADS), 0, s, t);
        if (t.draft && t.uniforms) hipLaunchKernelGGL(verify_left_kernel, dim3((unsigned)S, (unsigned)t.streams), dim3(VF_THREADS), 0, s, t);
        hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)t.streams), dim3(VF_THREADS), 0, s, t);
    }
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
