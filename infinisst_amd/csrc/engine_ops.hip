// Host side of libinfinisst_hip.so, part 4 of 4 (engine_internal.h): the per-kernel entry points of the C ABI (isst_op_*: parity tests drive every kernel
// through them) and the profiling hooks of bench.py.
#include "engine_internal.h"

extern "C" int64_t isst_op_packed_elems(int n_rows, int K) { return (int64_t)round_up(n_rows, 16) * K; }

extern "C" int isst_op_pack_weight(const uint16_t* w, uint16_t* packed, int n_rows, int K, int conv_k, void* hip_stream) {
    return launch_pack_weight(w, packed, n_rows, K, 0, 1, 0, conv_k, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_pack_gateup8(const uint16_t* gate, const uint16_t* up, uint16_t* packed, int ffn, int K, void* hip_stream) {
    if (!gate || !up || !packed) return ISST_ERR_ARG;
    const int rc = launch_pack_weight_half(gate, packed, ffn, K, 0, reinterpret_cast<hipStream_t>(hip_stream));
    return rc != ISST_OK ? rc : launch_pack_weight_half(up, packed, ffn, K, 1, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_gemm(const uint16_t* A, int64_t lda, const uint16_t* packed, const uint16_t* bias, const uint16_t* res, int64_t ldres,
                            void* out, int64_t ldo, int M, int N, int K, int n_valid, int epi, const uint16_t* norm_w, float norm_eps,
                            void* hip_stream) {
    GemmArgs g{};
    g.A = A; g.lda = lda; g.Wp = packed; g.bias = bias; g.res = res; g.ldres = ldres; g.out = out; g.ldo = ldo;
    g.M = M; g.N = round_up(N, 16); g.K = K; g.batch = 1; g.epi = epi; g.n_valid = n_valid;
    g.norm_w = norm_w; g.norm_eps = norm_eps;
    return launch_gemm(g, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_gemm_splitk_rmsnorm(const uint16_t* A, int64_t lda, const uint16_t* packed, uint16_t* x, const uint16_t* norm_w, uint16_t* out,
                                           float* slabs, int M, int N, int K, int ksplit, float norm_eps, void* hip_stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    if (N % 16 != 0) return ISST_ERR_ARG;
    GemmArgs g{};
    g.A = A; g.lda = lda; g.Wp = packed; g.out = slabs; g.ldo = N; g.out_batch = (long)M * N;
    g.M = M; g.N = N; g.K = K; g.batch = 1; g.epi = EPI_PARTIAL; g.n_valid = N; g.ksplit = ksplit;
    if (!gemm_mid_supported(g) && !gemm_tiled_supported(g)) return ISST_ERR_ARG;
    const int rc = launch_gemm(g, st);
    if (rc != ISST_OK) return rc;
    return launch_rmsnorm_reduce(slabs, (long)M * N, ksplit, x, N, norm_w, out, N, M, N, norm_eps, st);
}
extern "C" int isst_op_gemm_splitk_fused(const uint16_t* A, int64_t lda, const uint16_t* packed, uint16_t* x, float* slabs, float* ssq, int* tickets,
                                         int M, int N, int K, int ksplit, void* hip_stream) {
    if (N % 32 != 0 || !x || !slabs || !tickets) return ISST_ERR_ARG;
    GemmArgs g{};
    g.A = A; g.lda = lda; g.Wp = packed; g.out = slabs; g.ldo = N; g.out_batch = (long)M * N;
    g.M = M; g.N = N; g.K = K; g.batch = 1; g.epi = EPI_PARTIAL; g.n_valid = N; g.ksplit = ksplit;
    g.res = x; g.ldres = N; g.ssq = ssq; g.ssq_n = N / 32; g.tickets = tickets;
    if (!gemm_mid_supported(g)) return ISST_ERR_ARG;
    return launch_gemm_mid(g, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_gemm_splitk_plain(const uint16_t* A, int64_t lda, const uint16_t* packed, uint16_t* out, int64_t ldo, float* slabs, int* tickets,
                                         int M, int N, int K, int ksplit, const uint16_t* norm_w, float norm_eps, float* ssq_in, void* hip_stream) {
    if (N % 32 != 0 || !out || !slabs || !tickets || (norm_w && !ssq_in)) return ISST_ERR_ARG;
    GemmArgs g{};
    g.A = A; g.lda = lda; g.Wp = packed; g.out = slabs; g.ldo = N; g.out_batch = (long)M * N;
    g.M = M; g.N = N; g.K = K; g.batch = 1; g.epi = EPI_PARTIAL; g.n_valid = N; g.ksplit = ksplit;
    g.res = out; g.ldres = ldo; g.reduce_plain = 1; g.tickets = tickets;
    g.norm_w = norm_w; g.norm_eps = norm_eps; g.ssq = norm_w ? ssq_in : nullptr; g.ssq_n = norm_w ? K / 32 : 0;
    if (!gemm_mid_supported(g)) return ISST_ERR_ARG;
    return launch_gemm_mid(g, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_gemm_norm_ssq(const uint16_t* x, int64_t ldx, const uint16_t* packed, void* out, int64_t ldo, int M, int N, int K, int n_valid,
                                     int epi, const uint16_t* norm_w, float norm_eps, float* ssq, void* hip_stream) {
    if (!norm_w || !ssq) return ISST_ERR_ARG;
    GemmArgs g{};
    g.A = x; g.lda = ldx; g.Wp = packed; g.out = out; g.ldo = ldo;
    g.M = M; g.N = round_up(N, 16); g.K = K; g.batch = 1; g.epi = epi; g.n_valid = n_valid;
    g.norm_w = norm_w; g.norm_eps = norm_eps; g.ssq = ssq; g.ssq_n = K / 32;
    if (!gemm_mid_supported(g) && !gemm_wide_supported(g)) return ISST_ERR_ARG;
    return launch_gemm(g, reinterpret_cast<hipStream_t>(hip_stream));  // (gemm_mid.hip, or gemm_wide.hip for the widest projections from 33 rows on)
}
extern "C" int isst_op_gemm_splitk_layernorm(const uint16_t* A, int64_t lda, const uint16_t* packed, const uint16_t* bias, uint16_t* x,
                                             const uint16_t* ln_w, const uint16_t* ln_b, uint16_t* out, float* slabs, int M, int N, int K, int ksplit,
                                             float eps, void* hip_stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    if (N % 16 != 0 || !bias) return ISST_ERR_ARG;
    GemmArgs g{};
    g.A = A; g.lda = lda; g.Wp = packed; g.out = slabs; g.ldo = N; g.out_batch = (long)M * N;
    g.M = M; g.N = N; g.K = K; g.batch = 1; g.epi = EPI_PARTIAL; g.n_valid = N; g.ksplit = ksplit;
    if (!gemm_mid_supported(g) && !gemm_tiled_supported(g)) return ISST_ERR_ARG;
    const int rc = launch_gemm(g, st);
    if (rc != ISST_OK) return rc;
    return launch_layernorm_reduce(slabs, (long)M * N, ksplit, bias, x, N, ln_w, ln_b, out, N, M, N, eps, st);
}
extern "C" int isst_op_set_gemm_tuning(int waves_per_block, int ntiles_per_block) {
    gemm_set_tuning(waves_per_block, ntiles_per_block);
    return ISST_OK;
}
extern "C" int isst_profile_begin_rows(isst_handle* h, int rows_lo, int rows_hi) {
    if (!h || rows_lo < 1 || rows_hi < rows_lo) return h ? h->fail(ISST_ERR_ARG, "isst_profile_begin_rows: bad row range %d..%d", rows_lo, rows_hi) : ISST_ERR_ARG;
    h->prof_on = true;
    h->prof_used = 0;
    h->prof_rows_lo = rows_lo;
    h->prof_rows_hi = rows_hi;
    return ISST_OK;
}
extern "C" int isst_profile_begin(isst_handle* h) { return isst_profile_begin_rows(h, 1, 1); }
extern "C" int isst_profile_end(isst_handle* h, void* hip_stream, double* avg_us, int64_t* launches) {
    if (!h || !avg_us || !launches) return ISST_ERR_ARG;
    h->prof_on = false;
    HIPCHK(hipStreamSynchronize(reinterpret_cast<hipStream_t>(hip_stream)));
    double sum = 0.0;
    for (size_t i = 0; i + 1 < h->prof_used; i += 2) {
        float ms = 0.f;
        HIPCHK(hipEventElapsedTime(&ms, h->prof_ev[i], h->prof_ev[i + 1]));
        sum += ms * 1e3;
    }
    *launches = (int64_t)(h->prof_used / 2);
    *avg_us = *launches ? sum / *launches : 0.0;
    return ISST_OK;
}
extern "C" int isst_op_set_reduce_tuning(int rms_lf_rows, int ln_lf_rows) {
    reduce_set_tuning(rms_lf_rows, ln_lf_rows);
    return ISST_OK;
}
extern "C" int isst_op_set_attn_tuning(int target_workgroups) {
    llm_attn_set_tuning(target_workgroups);
    return ISST_OK;
}
extern "C" int isst_op_topk_rows(const float* scores, long ld, int vocab, int k, int rows, float* out_val, int* out_idx, void* hip_stream) {
    // test entry of beam.hip's per-row top-k (ties -> lowest index): out_val / out_idx are [rows][32] device arrays, the first k entries of a row are filled
    if (!scores || !out_val || !out_idx || rows < 1 || vocab < 1 || k < 1 || k > BEAM_TOPK || ld < vocab) return ISST_ERR_ARG;
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    float* cv = nullptr;
    int* ci = nullptr;
    if (hipMalloc(reinterpret_cast<void**>(&cv), sizeof(float) * (size_t)rows * 64 * BEAM_TOPK) != hipSuccess) return ISST_ERR_NOMEM;
    if (hipMalloc(reinterpret_cast<void**>(&ci), sizeof(int) * (size_t)rows * 64 * BEAM_TOPK) != hipSuccess) { (void)hipFree(cv); return ISST_ERR_NOMEM; }
    int rc = launch_topk_rows(scores, ld, vocab, k, cv, ci, out_val, out_idx, rows, st);
    if (hipStreamSynchronize(st) != hipSuccess && rc == ISST_OK) rc = ISST_ERR_HIP;
    (void)hipFree(cv);
    (void)hipFree(ci);
    return rc;
}
extern "C" int isst_op_layernorm(const uint16_t* x, const uint16_t* w, const uint16_t* b, uint16_t* out, int rows, int C, float eps, int gelu,
                                 void* hip_stream) {
    return launch_layernorm(x, C, w, b, out, C, rows, C, eps, gelu, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_rmsnorm(const uint16_t* x, const uint16_t* w, uint16_t* out, int rows, int D, float eps, void* hip_stream) {
    return launch_rmsnorm(x, D, nullptr, w, out, D, rows, D, eps, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_conv0(const uint16_t* audio, const uint16_t* w, const uint16_t* bias, const uint16_t* ln_w, const uint16_t* ln_b,
                             uint16_t* out, int T, int C, int k, int stride, void* hip_stream) {
    return launch_conv0(audio, 0, w, bias, ln_w, ln_b, out, 0, T, C, k, stride, 1, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_sample(float* logits, int vocab, const int* ids, int n_ids, const int* enc_ids, int n_enc, const int* suppress,
                              int n_suppress, float repetition_penalty, int ngram, int enc_ngram, int* out_token, void* hip_stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    SampleStream ss{n_ids, n_enc, 0, 0, 0};
    unsigned char* scratch = nullptr;  // [SampleStream | 64 floats | 64 ints]
    if (hipMalloc(reinterpret_cast<void**>(&scratch), 1024) != hipSuccess) return ISST_ERR_NOMEM;
    SampleStream* dss = reinterpret_cast<SampleStream*>(scratch);
    int rc = ISST_ERR_HIP;
    if (hipMemcpyAsync(dss, &ss, sizeof ss, hipMemcpyHostToDevice, st) == hipSuccess)
        rc = launch_sample(logits, vocab, vocab, dss, ids, enc_ids, suppress, n_suppress, repetition_penalty, ngram, enc_ngram, out_token,
                           reinterpret_cast<float*>(scratch + 256), reinterpret_cast<int*>(scratch + 512), 1, st);
    (void)hipStreamSynchronize(st);
    (void)hipFree(scratch);
    return rc;
}

extern "C" int isst_op_embed_splice(const int* ids, const int* speech_row, const uint16_t* table, const uint16_t* speech, uint16_t* out, int rows, int D,
                                    void* hip_stream) {
    if (!ids || !table || !out) return ISST_ERR_ARG;
    return launch_embed_splice(ids, speech_row, table, speech, out, rows, D, reinterpret_cast<hipStream_t>(hip_stream));
}

extern "C" int isst_op_enc_attention(const uint16_t* qkv, uint16_t* kring, uint16_t* vring, int ring_start, int prefix, const float* rope_cos,
                                     const float* rope_sin, int rope_round_each, uint16_t* out, int Q, int heads, int cap, int max_cache, int blocksize,
                                     void* hip_stream) {
    if (!qkv || !kring || !vring || !rope_cos || !rope_sin || !out || ring_start < 0 || ring_start >= cap || prefix < 0) return ISST_ERR_ARG;
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    EncStreamView hv{ring_start, prefix};
    EncStreamView* dv = nullptr;
    if (hipMalloc(reinterpret_cast<void**>(&dv), sizeof hv) != hipSuccess) return ISST_ERR_NOMEM;
    int rc = ISST_ERR_HIP;
    if (hipMemcpy(dv, &hv, sizeof hv, hipMemcpyHostToDevice) == hipSuccess)
        rc = launch_enc_attention(qkv, kring, vring, 0, dv, rope_cos, rope_sin, rope_round_each, out, 1, Q, heads, cap, max_cache, blocksize, st);
    if (hipStreamSynchronize(st) != hipSuccess && rc == ISST_OK) rc = ISST_ERR_HIP;
    (void)hipFree(dv);
    return rc;
}

extern "C" int isst_op_llm_attention(const uint16_t* qkv, int rows, int pos0, uint16_t* kpool, uint16_t* krpool, uint16_t* vpool, int heads, int kv_heads,
                                     int sys_cap, int ring_cap, int sys_len, int ring_start, const uint16_t* rope_cos, const uint16_t* rope_sin, int rot_keys,
                                     uint16_t* out, void* hip_stream) {
    if (!qkv || !kpool || !krpool || !vpool || !rope_cos || !rope_sin || !out || rows < 1 || pos0 < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads)
        return ISST_ERR_ARG;
    const int G = heads / kv_heads, slots = sys_cap + ring_cap;
    if ((G != 1 && G != 2 && G != 4) || slots % 64 || sys_cap % 16 || sys_len < 0 || sys_len > sys_cap || ring_start < 0 || ring_start >= ring_cap ||
        pos0 + rows - sys_len > ring_cap)
        return ISST_ERR_ARG;
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    LlmAttnDims d{};
    d.heads = heads; d.kv_heads = kv_heads; d.sys_cap = sys_cap; d.ring_cap = ring_cap; d.layer_stride = (long)kv_heads * slots * 128;
    LlmStreamView v{};
    v.sys_len = sys_len; v.ring_start = ring_start; v.kv_offset = 0; v.new_start = pos0; v.row0 = 0; v.rot_keys = rot_keys ? 1 : 0;
    const int gmax = LLM_ATTN_GROUP_ROWS(G);
    std::vector<int> row_stream(rows, 0), row_pos(rows);
    for (int r = 0; r < rows; ++r) row_pos[r] = pos0 + r;
    std::vector<int2> groups, units;
    for (int t = 0; t < rows; t += gmax) groups.push_back(make_int2(t, std::min(gmax, rows - t)));
    int max_unit_groups = 0;
    for (int g0 = 0; g0 < (int)groups.size(); g0 += LLM_PREFILL_UNIT_GROUPS) {
        units.push_back(make_int2(g0, std::min(LLM_PREFILL_UNIT_GROUPS, (int)groups.size() - g0)));
        max_unit_groups = std::max(max_unit_groups, units.back().y);
    }
    const size_t off_pos = sizeof(int) * rows, off_view = off_pos + sizeof(int) * rows, off_groups = (off_view + sizeof v + 15) / 16 * 16,
                 off_units = off_groups + sizeof(int2) * groups.size(), meta_bytes = off_units + sizeof(int2) * units.size();
    std::vector<unsigned char> hostm(meta_bytes);
    std::memcpy(hostm.data(), row_stream.data(), sizeof(int) * rows);
    std::memcpy(hostm.data() + off_pos, row_pos.data(), sizeof(int) * rows);
    std::memcpy(hostm.data() + off_view, &v, sizeof v);
    std::memcpy(hostm.data() + off_groups, groups.data(), sizeof(int2) * groups.size());
    std::memcpy(hostm.data() + off_units, units.data(), sizeof(int2) * units.size());
    unsigned char* meta = nullptr;
    float* partial = nullptr;
    if (hipMalloc(reinterpret_cast<void**>(&meta), meta_bytes) != hipSuccess) return ISST_ERR_NOMEM;
    if (hipMalloc(reinterpret_cast<void**>(&partial), sizeof(float) * (size_t)rows * heads * (slots / 64) * ATTN_SLAB) != hipSuccess) { (void)hipFree(meta); return ISST_ERR_NOMEM; }
    int rc = hipMemcpy(meta, hostm.data(), meta_bytes, hipMemcpyHostToDevice) == hipSuccess ? ISST_OK : ISST_ERR_HIP;
    const LlmStreamView* dv = reinterpret_cast<const LlmStreamView*>(meta + off_view);
    if (rc == ISST_OK && rot_keys && pos0 > 0) rc = launch_llm_rope_cache(dv, 1, rope_cos, rope_sin, kpool, krpool, d, 1, st);
    if (rc == ISST_OK) {
        LlmAttnOne one{};
        if (groups.size() == 1) { one.enabled = 1; one.grp = groups[0]; one.pos0 = pos0; one.pos_step = 1; one.v = v; }
        rc = launch_llm_attention(qkv, reinterpret_cast<const int*>(meta), reinterpret_cast<const int*>(meta + off_pos), dv,
                                  reinterpret_cast<const int2*>(meta + off_groups), (int)groups.size(), gmax, rope_cos, rope_sin, kpool, krpool, vpool, partial, out, d,
                                  0, rows, st, &one, reinterpret_cast<const int2*>(meta + off_units), (int)units.size(), max_unit_groups, 0);
    }
    if (hipStreamSynchronize(st) != hipSuccess && rc == ISST_OK) rc = ISST_ERR_HIP;
    (void)hipFree(meta);
    (void)hipFree(partial);
    return rc;
}

extern "C" int isst_op_splice_map(const int* ids, int len, int user_id, int assistant_id, int start_header_id, int n_features, int* row_src, int* n_rows) {
    if (!ids || len < 1 || !row_src || !n_rows || n_features < 0) return ISST_ERR_ARG;
    std::vector<int> desc;
    const int rc = splice_rows(ids, len, user_id, assistant_id, start_header_id, n_features, desc);
    if (rc != ISST_OK) return rc;
    *n_rows = (int)desc.size();  // <= len
    std::memcpy(row_src, desc.data(), sizeof(int) * desc.size());
    return ISST_OK;
}

// split-KV merge, as the combine launch and as the o_proj GEMV's A-staging prologue (parity test: the two must give the same bits)
extern "C" int isst_op_attn_combine(const float* partial, uint16_t* out, int heads, int rows, int n_splits, void* hip_stream) {
    if (!partial || !out) return ISST_ERR_ARG;
    return launch_llm_attn_combine(partial, out, heads, rows, n_splits, reinterpret_cast<hipStream_t>(hip_stream));
}
extern "C" int isst_op_gemm_attn_merge(const float* partial, int n_splits, const uint16_t* packed, const uint16_t* res, int64_t ldres, uint16_t* out,
                                       int64_t ldo, int M, int N, int K, void* hip_stream) {
    if (!partial || !packed || !out) return ISST_ERR_ARG;
    GemmArgs g{};
    g.lda = K; g.Wp = packed; g.res = res; g.ldres = ldres; g.out = out; g.ldo = ldo;
    if (!res) return ISST_ERR_ARG;
    g.M = M; g.N = round_up(N, 16); g.K = K; g.batch = 1; g.epi = EPI_RES; g.n_valid = N;
    g.attn_partial = partial; g.attn_splits = n_splits;
    return launch_gemm(g, reinterpret_cast<hipStream_t>(hip_stream));
}

// ---- a decode step of many streams over one prompt (prefix_attn.hip, lora.hip, verify.hip) ----
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool prefix_attention_ok(const isst_prefix_attn* a) {
    if (!a || a->rows < 0 || a->seqs < 0 || a->max_rows < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || (a->head_dim != 64 && a->head_dim != 128) ||
        a->prefix_len < 0 || a->tail_cap < 0 || !(a->scale > 0.f) || !(a->scale < INFINITY))
        return false;
    if (a->heads > (1 << 15) || (int64_t)a->rows * a->heads > (1 << 26) || (int64_t)a->seqs * a->kv_heads > (1 << 22) || (a->rows > 0 && a->seqs < 1)) return false;
    if (!a->row_starts && a->seqs > 0 && a->rows % a->seqs) return false;
    if (a->rows == 0) return true;
    if (!a->q || !a->out || !a->tail_lens || !aligned16(a->q) || !aligned16(a->out)) return false;
    int64_t strides = a->q_row | a->q_head | a->out_row | a->out_head;
    if (a->prefix_len > 0) {
        if (!a->k_prefix || !a->v_prefix || !aligned16(a->k_prefix) || !aligned16(a->v_prefix)) return false;
        strides |= a->kp_head | a->kp_key | a->vp_head | a->vp_key;
    }
    if (a->tail_cap > 0) {
        if (!a->k_tail || !a->v_tail || !aligned16(a->k_tail) || !aligned16(a->v_tail)) return false;
        strides |= a->kt_seq | a->kt_head | a->kt_key | a->vt_seq | a->vt_head | a->vt_key;
    }
    if (strides & 7) return false;
    for (const int64_t key : {a->kp_key, a->vp_key, a->kt_key, a->vt_key})  // (32-bit offsets inside a tile of 32 keys)
        if (key < 0 || key > (1 << 24)) return false;
    // two outputs never share memory: the heads of a row lie together, or the rows of a head
    const bool one_head = a->heads == 1, one_row = a->rows == 1;
    if ((!one_head && a->out_head < a->head_dim) || (!one_row && a->out_row < a->head_dim)) return false;
    return one_head || one_row || (a->out_row - a->head_dim) / a->out_head >= a->heads - 1 || (a->out_head - a->head_dim) / a->out_row >= a->rows - 1;
}
extern "C" int64_t isst_op_prefix_attention_workspace(const isst_prefix_attn* a) { return prefix_attention_ok(a) ? (a->rows ? prefix_attention_workspace(*a) : 0) : ISST_ERR_ARG; }
extern "C" int isst_op_prefix_attention(const isst_prefix_attn* a, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    if (!prefix_attention_ok(a)) return ISST_ERR_ARG;
    if (a->rows == 0) return ISST_OK;
    const int64_t need = prefix_attention_workspace(*a);
    if (need > 0 && (!workspace || !aligned16(workspace))) return ISST_ERR_ARG;
    if (workspace_bytes < need) return ISST_ERR_NOMEM;
    return launch_prefix_attention(*a, workspace, reinterpret_cast<hipStream_t>(hip_stream));
}

// K slices of the base product: fp32 slabs through the many-row kernels, the raw accumulator through the register-A one where they do not run
static GemmArgs lora_base_args(const uint16_t* A, int64_t lda, const uint16_t* packed, float* base, int M, int N, int K) {
    GemmArgs g{};
    g.A = A; g.lda = lda; g.Wp = packed; g.out = base; g.N = round_up(N, 16); g.ldo = g.N; g.out_batch = (long)M * g.N;
    g.M = M; g.K = K; g.batch = 1; g.n_valid = N;
    g.epi = EPI_PARTIAL;
    // as many K slices as give every compute unit a workgroup of that kernel, in one round (the base in us, slices 1 / 2 / 4: 64 rows of 4096 x 6144 23 / 18 / 23, 1408 rows of 4096 x 4096
    // 78 / 52 / 61; slices 2 / 4 / 8: 320 rows of 14336 x 4096 120 / 72 / 50)
    g.ksplit = 1;
    if (M > 64 && !gemm_dense_would_run(M, g.N, K)) g.ksplit = pick_ksplit(K, g.N, M, 1L << 28);
    else if (M > 12) {
        const int blocks = M > 64 ? (g.N + 255) / 256 * ((M + 255) / 256) : (g.N + 63) / 64, step = M > 64 ? 64 : 256, least = M > 64 ? 16 : 1;
        for (int s = 2; s <= (M > 64 ? 8 : 4) && blocks * s <= 256 && K % (step * s) == 0 && K / (step * s) >= least; s *= 2) g.ksplit = s;
    }
    if (gemm_mid_supported(g) || gemm_tiled_supported(g)) return g;
    g.ksplit = 1;
    if (gemm_mid_supported(g) || gemm_tiled_supported(g)) return g;
    g.epi = EPI_RAW;
    return g;
}
static bool lora_ok(int M, int N, int K, int rank, int n_adapters) {
    return M >= 0 && N >= 1 && N <= (1 << 21) && K >= 32 && K % 32 == 0 && K <= (1 << 24) && rank >= 8 && rank <= 128 && rank % 8 == 0 && n_adapters >= 1 &&
           (int64_t)M * N < (1L << 30) && (int64_t)M * K < (1L << 29);
}
extern "C" int64_t isst_op_gemm_lora_workspace(int M, int N, int K, int rank, int n_adapters) {
    if (!lora_ok(M, N, K, rank, n_adapters)) return ISST_ERR_ARG;
    const GemmArgs g = lora_base_args(nullptr, K, nullptr, nullptr, M, N, K);
    return ((int64_t)g.ksplit * M * g.N + lora_t_floats(M, N, K, rank, n_adapters)) * (int64_t)sizeof(float);
}
extern "C" int isst_op_gemm_lora(const uint16_t* A, int64_t lda, const uint16_t* packed, const uint16_t* down, const uint16_t* up, const float* scales,
                                 const int* row_adapter, int n_adapters, int rank, uint16_t* out, int64_t ldo, int M, int N, int K, void* workspace,
                                 int64_t workspace_bytes, void* hip_stream) {
    if (!lora_ok(M, N, K, rank, n_adapters)) return ISST_ERR_ARG;
    if (M == 0) return ISST_OK;
    if (!A || !packed || !down || !up || !scales || !row_adapter || !out || !workspace || lda < K || lda % 8 || (int64_t)M * lda >= (1L << 29) || ldo < N || !aligned16(A) ||
        !aligned16(packed) || !aligned16(down) || !aligned16(up) || !aligned16(workspace))
        return ISST_ERR_ARG;
    if (workspace_bytes < isst_op_gemm_lora_workspace(M, N, K, rank, n_adapters)) return ISST_ERR_NOMEM;
    hipStream_t st = reinterpret_cast<hipStream_t>(hip_stream);
    const GemmArgs g = lora_base_args(A, lda, packed, static_cast<float*>(workspace), M, N, K);
    LoraArgs l{};
    l.A = A; l.lda = lda; l.down = down; l.up = up; l.scales = scales; l.row_adapter = row_adapter;
    l.base = static_cast<const float*>(workspace); l.ld_base = g.N; l.slabs = g.ksplit;
    l.t = static_cast<float*>(workspace) + (int64_t)g.ksplit * M * g.N;
    l.out = out; l.ldo = ldo; l.M = M; l.N = N; l.K = K; l.rank = rank; l.n_adapters = n_adapters;
    int rc = launch_lora_down(l, st);
    // the kernel behind EPI_RAW has 64 rows a workgroup along the grid's second dimension, which ends at 65536 (depths that are no multiple of 64: M goes up to 2^24)
    const int rows = g.epi == EPI_RAW ? 64 * 65535 : M;
    for (int m0 = 0; rc == ISST_OK && m0 < M; m0 += rows) {
        GemmArgs part = g;
        part.A += (int64_t)m0 * lda;
        part.out = static_cast<float*>(workspace) + (int64_t)m0 * g.N;
        part.M = M - m0 < rows ? M - m0 : rows;
        rc = launch_gemm(part, st);
    }
    if (rc == ISST_OK) rc = launch_lora_up(l, st);
    return rc;
}

static bool verify_ok(int streams, int max_drafts, int vocab) {
    return streams >= 0 && max_drafts >= 0 && max_drafts < (1 << 14) && vocab >= 1 && vocab <= (1 << 30) && streams < (1 << 24);
}
extern "C" int64_t isst_op_verify_drafts_workspace(int streams, int max_drafts, int vocab) {
    return verify_ok(streams, max_drafts, vocab) ? verify_workspace(streams, max_drafts, vocab) : ISST_ERR_ARG;
}
extern "C" int isst_op_verify_drafts(const float* target, int64_t target_stream, int64_t target_row, const float* draft_scores, int64_t draft_stream, int64_t draft_row,
                                     const int* drafts, const int* n_drafts, const double* uniforms, int streams, int max_drafts, int vocab, int* tokens, int* counts,
                                     void* workspace, int64_t workspace_bytes, void* hip_stream) {
    if (!verify_ok(streams, max_drafts, vocab)) return ISST_ERR_ARG;
    if (streams == 0) return ISST_OK;
    if (!target || (max_drafts > 0 && !drafts) || !tokens || !counts || !workspace || !aligned16(workspace) || target_stream < 0 || target_row < 0 || draft_stream < 0 || draft_row < 0 ||
        ((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft_scores) | reinterpret_cast<uintptr_t>(drafts) | reinterpret_cast<uintptr_t>(n_drafts) |
          reinterpret_cast<uintptr_t>(tokens) | reinterpret_cast<uintptr_t>(counts)) & 3) || (reinterpret_cast<uintptr_t>(uniforms) & 7))
        return ISST_ERR_ARG;
    if (workspace_bytes < verify_workspace(streams, max_drafts, vocab)) return ISST_ERR_NOMEM;
    VerifyArgs v{};
    v.target = target; v.target_stream = target_stream; v.target_row = target_row;
    v.draft = max_drafts > 0 && uniforms ? draft_scores : nullptr; v.draft_stream = draft_stream; v.draft_row = draft_row;
    v.drafts = drafts; v.n_drafts = n_drafts; v.uniforms = uniforms; v.streams = streams; v.max_drafts = max_drafts; v.vocab = vocab;
    v.tokens = tokens; v.counts = counts; v.workspace = workspace;
    return launch_verify(v, reinterpret_cast<hipStream_t>(hip_stream));
}
