// Verification of drafted tokens (gfx950): accept draft x_i while u_i q_i(x_i) < p_i(x_i), then draw from max(p_i - q_i, 0) or, with every draft accepted, from p_n.
// p, q = softmax of fp32 score rows.  Everything behind the scores is in 64 bits: the outcome of a comparison or of a draw must not depend on the order of a sum, and with
// 32-bit probabilities the borders of the inverse CDF move by ~1e-8 each -- over 128 k of them one draw in a thousand would land elsewhere.
//
// Launch 1 reads every score row once, a workgroup per slice of VF_SLICE entries (maximum and its first index, or sum of exponentials); its floor is that read, and most of
// the 64-bit exponentials hides behind it.  Drafts with scores need two more: who decides (a workgroup per stream), and what a refused draft leaves over, slice by slice.  The last
// launch takes one workgroup per stream: find the slice that the draw falls into from the slice sums, walk that slice.
// Measured, rows of 128263: 64 streams x 4 drafts with scores 59 us (263 MB: 4.5 TB/s) + decide 4.8 + left over 15.1 + draw 6.7; one stream without scores 6.3 + 7.0, latency all of it (in cycles
// of the draw: decide 5400, find the slice 3300, its weights 3200, walk 2600).
#include "common.h"
#include "kernels.h"

#define VF_THREADS 256
#define VF_PER 16                          // entries of a lane
#define VF_SLICE (VF_THREADS * VF_PER)
#define VF_ROWS 32                         // drafts that are decided at a time
#define VF_DRAW 512                       // threads of the workgroup that decides and draws for a stream: its time is latency, and the walk through a slice takes eight exponentials a lane

struct VerifyStat { double sum; float max; int at; };  // of a slice: sum of exp(score - max), max (NaN: a NaN or +inf among the scores), the maximum's first index

typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));  // (rows start anywhere)

// exp(d) for -700 <= d <= 0: 2^k exp(r), k the nearest whole number to d / ln 2 (added to 1.5 2^52, where it is the low word), |r| <= ln 2 / 2, the polynomial of degree 10 through exp at the
// Chebyshev nodes of that interval.  Relative error (checked against 60 digits on 4001 points): 4.3e-16 of the polynomial, i.e. two roundings, and 2.4e-17 |k| of the one-term reduction -- 1.7e-15
// down to d = -40; over 128 k borders of an inverse CDF one draw in 10^9 could land elsewhere for it.  The score read is bound by these instructions, a 64-bit multiply-add an entry is 2.4 us of the
// 84 that 64 streams x 4 drafts with scores take (degree 8, 1.05e-12: 80 -- but then uniforms 1e-12 beside a probability are decided wrongly, relative to it).
__device__ __forceinline__ double exp_core(double d) {
    const double t = fma(d, 1.4426950408889634074, 0x1.8p52), k = t - 0x1.8p52, r = fma(-k, 0.69314718055994530942, d);
    double p = 2.7626426376580335e-07;
    p = fma(p, r, 2.7640263790318923e-06); p = fma(p, r, 2.4801504180837137e-05); p = fma(p, r, 0.00019841170070971308); p = fma(p, r, 0.0013888888932619635); p = fma(p, r, 0.008333333385825085);
    p = fma(p, r, 0.04166666666657277); p = fma(p, r, 0.16666666666553953); p = fma(p, r, 0.5000000000000006); p = fma(p, r, 1.0000000000000069); p = fma(p, r, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}
// ... for any d <= 0; under -700 and for NaN (-inf less -inf): 0
__device__ __forceinline__ double exp_le0(double d) { return d >= -700.0 ? exp_core(d) : 0.0; }
// 64-bit reductions over lanes on DPP (as common.h's 32-bit ones): the rows of 16 lanes inside the vector ALU, the four rows by v_readlane -- a tree of ds_bpermute pairs is 0.7 us of latency
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {  // (lanes without a source: 0)
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true), hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true);
    return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double lane_d(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double row_sum_d(double v) {  // of the 16 lanes of a row, in each of them
    v += dpp_d<0xb1>(v);
    v += dpp_d<0x4e>(v);
    v += dpp_d<0x124>(v);
    v += dpp_d<0x128>(v);
    return v;
}
__device__ __forceinline__ double half_sum_d(double v) {  // of the 32 lanes of a half wave
    v = row_sum_d(v);
    const double a = lane_d(v, 0) + lane_d(v, 16), b = lane_d(v, 32) + lane_d(v, 48);
    return (threadIdx.x & 32) ? b : a;
}
__device__ __forceinline__ double wave_sum_d(double v) {
    v = row_sum_d(v);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}
// sum over this lane and the lanes before it
__device__ __forceinline__ double wave_scan_d(double v) {
    v += dpp_d<0x111>(v);
    v += dpp_d<0x112>(v);
    v += dpp_d<0x114>(v);
    v += dpp_d<0x118>(v);
    const double r0 = lane_d(v, 15), r1 = r0 + lane_d(v, 31), r2 = r1 + lane_d(v, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return row == 0 ? v : v + (row == 1 ? r0 : row == 2 ? r1 : r2);
}
// the (value, lowest index) maximum of the 32 lanes of a half wave
__device__ __forceinline__ void half_argmax(float& m, int& at) {
    float v = m;
    v = fmaxf(v, __int_as_float(dpp_take<0xb1>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(dpp_take<0x4e>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(dpp_take<0x124>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(dpp_take<0x128>(__float_as_int(v))));
    auto lane_f = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
    const float a = fmaxf(lane_f(0), lane_f(16)), b = fmaxf(lane_f(32), lane_f(48));
    v = (threadIdx.x & 32) ? b : a;
    int i = m == v ? at : 0x7fffffff;
    i = min(i, dpp_take<0xb1>(i));
    i = min(i, dpp_take<0x4e>(i));
    i = min(i, dpp_take<0x124>(i));
    i = min(i, dpp_take<0x128>(i));
    const int ia = min(__builtin_amdgcn_readlane(i, 0), __builtin_amdgcn_readlane(i, 16)), ib = min(__builtin_amdgcn_readlane(i, 32), __builtin_amdgcn_readlane(i, 48));
    m = v;
    at = (threadIdx.x & 32) ? ib : ia;
}
__device__ __forceinline__ int slices(int vocab) { return (vocab + VF_SLICE - 1) / VF_SLICE; }
__device__ __forceinline__ int rows_of(const VerifyArgs& g) { return g.max_drafts + 1 + (g.draft ? g.max_drafts : 0); }
__device__ __forceinline__ const VerifyStat* stats_of(const VerifyArgs& g, int b, int row) {
    return static_cast<const VerifyStat*>(g.workspace) + ((long)b * rows_of(g) + row) * slices(g.vocab);
}
// behind the statistics, per stream: what a refused draft with scores leaves over, [slices]; or, of drafts without, the sum of the draft's slice without the draft, [max_drafts]
__device__ __forceinline__ int rest_of(const VerifyArgs& g) { return g.draft ? slices(g.vocab) : g.max_drafts; }
__device__ __forceinline__ double* left_of(const VerifyArgs& g, int b) {
    return reinterpret_cast<double*>(static_cast<VerifyStat*>(g.workspace) + (long)g.streams * rows_of(g) * slices(g.vocab)) + (long)b * rest_of(g);
}
__device__ __forceinline__ const float* target_row(const VerifyArgs& g, int b, int i) { return g.target + b * g.target_stream + i * g.target_row; }
__device__ __forceinline__ const float* draft_row(const VerifyArgs& g, int b, int i) { return g.draft + b * g.draft_stream + i * g.draft_row; }

// grid (slices, score rows)
template <bool GREEDY>
__global__ __launch_bounds__(VF_THREADS) void verify_stats_kernel(VerifyArgs g) {
    __shared__ VerifyStat part[VF_THREADS / 64];
    __shared__ double rests[VF_THREADS / 64];
    const int tid = threadIdx.x, wave = tid >> 6, rows_t = g.max_drafts + 1, per = rows_of(g);
    const int b = blockIdx.y / per, i = blockIdx.y % per, lo = blockIdx.x * VF_SLICE;
    if (g.n_drafts && (i < rows_t ? i : i - rows_t + 1) > g.n_drafts[b]) return;  // (a row behind the stream's drafts)
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
        if (!GREEDY) m = fmaxf(m, s[k]);
        else if (s[k] > m) { m = s[k]; at = lo + ((k >> 2) * VF_THREADS + tid) * 4 + (k & 3); }
    }
    double sum = 0.0, rest = 0.0;
    int x_at = -1;  // the row's draft, where it comes without scores and lies in this slice
    if constexpr (GREEDY) {
        wave_argmax_all(m, at);
    } else {
        m = wave_max_all(m);
#pragma unroll
        for (int k = 0; k < VF_PER; ++k) sum += exp_core(fmax((double)s[k] - (double)m, -700.0));  // (1e-304 for a removed entry: not one bit of a sum that is 1 or more)
        sum = wave_sum_d(sum);
        if (!g.draft && i < g.max_drafts) {
            const int xi = g.drafts[(long)b * g.max_drafts + i];
            if (xi >= lo && xi - lo < VF_SLICE) x_at = xi;
        }
        if (x_at >= 0) {
#pragma unroll
            for (int k = 0; k < VF_PER; ++k) rest += lo + ((k >> 2) * VF_THREADS + tid) * 4 + (k & 3) == x_at ? 0.0 : exp_le0((double)s[k] - (double)m);
            rest = wave_sum_d(rest);
        }
    }
    bad = __any(bad);
    if ((tid & 63) == 0) { part[wave] = {sum, bad ? NAN : m, at}; rests[wave] = rest; }
    __syncthreads();
    if (tid == 0) {
        VerifyStat t = part[0];
        double r = rests[0];
        for (int w = 1; w < VF_THREADS / 64; ++w) {
            const VerifyStat o = part[w];
            if (!(t.max == t.max) || !(o.max == o.max)) { t.max = NAN; continue; }
            const float M = fmaxf(t.max, o.max);
            const double et = exp_le0((double)t.max - (double)M), eo = exp_le0((double)o.max - (double)M);
            t.sum = t.sum * et + o.sum * eo;
            r = r * et + rests[w] * eo;
            if (o.max > t.max) t.at = o.at;  // (equal: the lower index is the earlier one -- below)
            else if (o.max == t.max) t.at = min(t.at, o.at);
            t.max = M;
        }
        static_cast<VerifyStat*>(g.workspace)[(long)blockIdx.y * gridDim.x + blockIdx.x] = t;
        if (x_at >= 0) left_of(g, b)[i] = r;
    }
}

// one row's statistics from its slices, by the 32 lanes of a half wave (row < 0: none of its business), in each of them; max = NaN: no distribution
__device__ __forceinline__ VerifyStat merge_row(const VerifyArgs& g, int b, int row) {
    const VerifyStat* st = stats_of(g, b, max(row, 0));
    const int S = row < 0 ? 0 : slices(g.vocab), lane = threadIdx.x & 31;
    VerifyStat t = {0.0, -INFINITY, 0x7fffffff};
    bool bad = false;
    for (int s = lane; s < S; s += 32) {
        const VerifyStat o = st[s];
        bad |= !(o.max == o.max);
        const float M = fmaxf(t.max, o.max);
        t.sum = t.sum * exp_le0((double)t.max - (double)M) + o.sum * exp_le0((double)o.max - (double)M);
        if (o.max > t.max) t.at = o.at;  // (slices come in index order: on equality the earlier one stays)
        t.max = M;
    }
    float M = t.max;
    int at = t.at;
    half_argmax(M, at);
    t.sum = half_sum_d(t.sum * exp_le0((double)t.max - (double)M));
    const unsigned long long bads = __ballot(bad);
    t.max = ((threadIdx.x & 32) ? bads >> 32 : bads & 0xffffffffull) || M == -INFINITY ? NAN : M;
    t.at = at;
    return t;
}

struct Decision {
    int accepted, n;  // accepted < 0: no answer
    VerifyStat p, q;  // of the row that decides (q: of the refused draft's scores)
};
// by the whole workgroup of VF_DRAW threads, the same in every thread
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
        const int looks = g.draft ? 2 * cnt + 1 : cnt + 1;
        for (int k0 = 2 * wave; k0 < looks; k0 += VF_DRAW / 32) {
            const int k = k0 + ((tid >> 5) & 1);
            const VerifyStat t = merge_row(g, b, k >= looks ? -1 : k <= cnt ? i0 + k : K + 1 + i0 + k - cnt - 1);
            if ((tid & 31) == 0 && k < looks) {
                if (k <= cnt) sp[k] = t;
                else sq[k - cnt - 1] = t;
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
// the lane's entries lo + PER tid .. of the slice
template <int PER>
__device__ __forceinline__ void weights(const VerifyArgs& g, int b, const Decision& d, int kind, int lo, double (&w)[PER]) {
    const int i = d.accepted, v0 = lo + PER * threadIdx.x, xi = kind == 1 ? g.drafts[(long)b * g.max_drafts + i] : -1;
    const float *t = target_row(g, b, i), *q = kind == 0 ? draft_row(g, b, i) : t;
    const double inv_p = 1.0 / d.p.sum, inv_q = kind == 0 ? 1.0 / d.q.sum : 0.0;
    float ts[PER], qs[PER];
#pragma unroll
    for (int k = 0; k < PER; k += 4) {
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
    for (int k = 0; k < PER; ++k) w[k] = weight(kind, d, ts[k], qs[k], v0 + k == xi, inv_p, inv_q);
}
// inclusive sum over the workgroup's threads in thread order, and the total
template <int THREADS>
__device__ __forceinline__ double block_scan(double v, double& total) {
    __shared__ double wsum[THREADS / 64];
    const int wave = threadIdx.x >> 6;
    v = wave_scan_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) wsum[wave] = v;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += wsum[w];
        total += wsum[w];
    }
    return before + v;
}
__device__ __forceinline__ double slice_sum(const VerifyArgs& g, int b, const Decision& d, int kind, int lo) {
    double w[VF_PER], mine = 0.0, total;
    weights<VF_PER>(g, b, d, kind, lo, w);
#pragma unroll
    for (int k = 0; k < VF_PER; ++k) mine += w[k];
    block_scan<VF_THREADS>(mine, total);
    return total;
}

__device__ __forceinline__ Decision* decision_of(const VerifyArgs& g, int b) { return reinterpret_cast<Decision*>(left_of(g, g.streams)) + b; }
__global__ __launch_bounds__(VF_DRAW) void verify_decide_kernel(VerifyArgs g) {
    const Decision d = decide(g, blockIdx.x);
    if (threadIdx.x == 0) *decision_of(g, blockIdx.x) = d;
}

// grid (slices, streams): what a refused draft with scores leaves over
__global__ __launch_bounds__(VF_THREADS) void verify_left_kernel(VerifyArgs g) {
    const Decision d = *decision_of(g, blockIdx.y);
    if (d.accepted < 0 || d.accepted == d.n) return;
    const double s = slice_sum(g, blockIdx.y, d, 0, blockIdx.x * VF_SLICE);
    if (threadIdx.x == 0) left_of(g, blockIdx.y)[blockIdx.x] = s;
}

// one workgroup per stream
template <bool DECIDED>
__global__ __launch_bounds__(VF_DRAW) void verify_draw_kernel(VerifyArgs g) {
    constexpr int PER = VF_SLICE / VF_DRAW;
    __shared__ int s_slice, s_live, s_at[VF_DRAW / 64], s_last[VF_DRAW / 64];
    __shared__ double s_before, s_total;
    const int b = blockIdx.x, tid = threadIdx.x, K = g.max_drafts, S = slices(g.vocab);
    const Decision d = DECIDED ? *decision_of(g, b) : decide(g, b);
    int pick = -1;
    bool bad = d.accepted < 0;
    if (!bad && !g.uniforms) pick = d.p.at;
    if (!bad && g.uniforms) {
        const double u = g.uniforms[(long)b * (K + 1) + K];
        bad = !(u >= 0.0 && u < 1.0);
        const VerifyStat* st = stats_of(g, b, d.accepted);
        for (int kind = bad ? 3 : d.accepted == d.n ? 2 : g.draft ? 0 : 1; kind < 3; kind = 2) {
            const int xs = kind == 1 ? g.drafts[(long)b * K + d.accepted] / VF_SLICE : -1;  // (the slice that the draft is taken out of)
            auto of_slice = [&](int s) {
                if (kind == 0) return left_of(g, b)[s];
                return (s == xs ? left_of(g, b)[d.accepted] : st[s].sum) * exp_le0((double)st[s].max - (double)d.p.max) / d.p.sum;
            };
            if (tid < 64) {  // total, then the slice whose running sum first exceeds u total (none, by rounding: the last one that holds anything)
                double total = 0.0;
                const double head = tid < S ? of_slice(tid) : 0.0;
                for (int s0 = 0; s0 < S; s0 += 64) total += wave_sum_d(s0 == 0 ? head : s0 + tid < S ? of_slice(s0 + tid) : 0.0);
                int slice = -1, live = -1;
                double before = 0.0, cum = 0.0;
                for (int s0 = 0; s0 < S && slice < 0; s0 += 64) {
                    const double v = s0 == 0 ? head : s0 + tid < S ? of_slice(s0 + tid) : 0.0, c = cum + wave_scan_d(v);
                    const unsigned long long hit = __ballot(v > 0.0 && c > u * total), any = __ballot(v > 0.0);
                    const int at = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : -1;
                    if (at >= 0) { live = s0 + at; before = lane_d(c - v, __builtin_amdgcn_readfirstlane(at)); }
                    if (hit) slice = live;
                    cum = lane_d(c, 63);
                }
                if (tid == 0) { s_slice = slice; s_live = live; s_before = before; s_total = total; }
            }
            __syncthreads();
            const double total = s_total, goal = s_slice < 0 ? INFINITY : u * total;
            const int slice = s_live;
            if (!(total > 0.0) || slice < 0) {  // nothing left over: the row itself
                __syncthreads();
                if (kind == 2) break;
                continue;
            }
            double w[PER], mine = 0.0, all;
            weights<PER>(g, b, d, kind, slice * VF_SLICE, w);
#pragma unroll
            for (int k = 0; k < PER; ++k) mine += w[k];
            double cum = s_before + (block_scan<VF_DRAW>(mine, all) - mine);
            int at = 0x7fffffff, last = -1;
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                if (!(w[k] > 0.0)) continue;
                cum += w[k];
                last = slice * VF_SLICE + PER * tid + k;
                if (cum > goal && at == 0x7fffffff) at = last;
            }
            // the first thread that passes the goal, or the last that holds anything (threads are in index order; atomics on one address of LDS took 3 us here)
            const unsigned long long hits = __ballot(at != 0x7fffffff), lives = __ballot(last >= 0);
            const int first = __builtin_amdgcn_readlane(at, hits ? __builtin_ctzll(hits) : 0), end = __builtin_amdgcn_readlane(last, lives ? 63 - __builtin_clzll(lives) : 0);
            if ((tid & 63) == 0) { s_at[tid >> 6] = first; s_last[tid >> 6] = end; }
            __syncthreads();
            at = 0x7fffffff; last = -1;
#pragma unroll
            for (int w = 0; w < VF_DRAW / 64; ++w) { at = min(at, s_at[w]); last = max(last, s_last[w]); }
            pick = at != 0x7fffffff ? at : last;
            break;
        }
    }
    bad |= pick < 0;
    for (int k = tid; k <= K; k += VF_DRAW) g.tokens[(long)b * (K + 1) + k] = bad ? -1 : k < d.accepted ? g.drafts[(long)b * K + k] : k == d.accepted ? pick : -1;
    if (tid == 0) g.counts[b] = bad ? -1 : d.accepted + 1;
}

static int64_t n_slices(int vocab) { return ((int64_t)vocab + VF_SLICE - 1) / VF_SLICE; }
int64_t verify_workspace(int streams, int max_drafts, int vocab) {
    const int64_t rest = n_slices(vocab) > max_drafts ? n_slices(vocab) : max_drafts;
    return streams * (n_slices(vocab) * (2 * (int64_t)max_drafts + 1) * (int64_t)sizeof(VerifyStat) + rest * (int64_t)sizeof(double) + (int64_t)sizeof(Decision));
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
        const dim3 grid((unsigned)S, (unsigned)(t.streams * per)), block(VF_THREADS), per_stream((unsigned)t.streams), draw(VF_DRAW);
        if (!t.uniforms) hipLaunchKernelGGL(verify_stats_kernel<true>, grid, block, 0, s, t);
        else hipLaunchKernelGGL(verify_stats_kernel<false>, grid, block, 0, s, t);
        if (t.draft) {
            hipLaunchKernelGGL(verify_decide_kernel, per_stream, draw, 0, s, t);
            hipLaunchKernelGGL(verify_left_kernel, dim3((unsigned)S, (unsigned)t.streams), block, 0, s, t);
            hipLaunchKernelGGL(verify_draw_kernel<true>, per_stream, draw, 0, s, t);
        } else {
            hipLaunchKernelGGL(verify_draw_kernel<false>, per_stream, draw, 0, s, t);
        }
    }
    return hipGetLastError() == hipSuccess ? ISST_OK : ISST_ERR_HIP;
}
