"""Cases of the decode-step operators that serve many streams from one set of weights and one prompt:

  prefix_attention  attention of a batch whose sequences share one long prefix (a system prompt with its glossary, the common
                    history of beam hypotheses) in front of keys of their own; the prefix is read once for the whole batch
  gemm_lora         a shared projection with a low-rank adapter of its own per row (one adapter per language pair)
  verify_drafts     acceptance of drafted tokens against the model's scores at given uniforms, and the draw that follows

`run` computes them in elementary torch operations, or (own = True) by the library's entry points on the same inputs."""
import math

import torch

own = False

DEV = "cuda"
LLM = dict(heads=32, kv_heads=8, dim=128)  # the decoder of the full configuration
VOCAB = 128263
QKV, O, DOWN = (4096, 6144), (4096, 4096), (14336, 4096)  # (in, out) of its fused q/k/v, output and down projections


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # four beams of one stream, a few tokens into a chunk, over the cache they share: the smallest call of a decode step
        dict(name="attn_beams", op="attn", seqs=4, rows=1, prefix=1000, tail=9, ragged=False, **LLM),
        # 64 streams, one new token each: a system prompt with a glossary in front of histories of 23 to 1000 tokens
        dict(name="attn_decode", op="attn", seqs=64, rows=1, prefix=4093, tail=1000, ragged=True, **LLM),
        # the same with five rows a stream, as a pass that checks four drafted tokens has them
        dict(name="attn_drafts", op="attn", seqs=64, rows=5, prefix=8192, tail=517, ragged=False, **LLM),
        # the prompt pass of a tick: 1 to 22 new rows a stream
        dict(name="attn_prompts", op="attn", seqs=64, rows=22, prefix=8001, tail=1022, ragged=True, **LLM),
        # heads of 64, one key head per query head (the encoder's layout)
        dict(name="attn_heads64", op="attn", seqs=33, rows=3, prefix=2047, tail=129, ragged=True, heads=16, kv_heads=16, dim=64),
        # one stream's decode row through q/k/v: latency
        dict(name="lora_row", op="lora", rows=1, K=QKV[0], N=QKV[1], rank=16, adapters=8, spread="runs"),
        # 64 streams, every one with an adapter of its own
        dict(name="lora_decode", op="lora", rows=64, K=QKV[0], N=QKV[1], rank=16, adapters=64, spread="mixed"),
        # five rows a stream (drafts), rank 64, the deep projection
        dict(name="lora_drafts", op="lora", rows=320, K=DOWN[0], N=DOWN[1], rank=64, adapters=12, spread="runs"),
        # the prompt pass of 64 streams: runs of 22 rows
        dict(name="lora_prompts", op="lora", rows=1408, K=O[0], N=O[1], rank=32, adapters=16, spread="runs"),
        # one stream whose draft is its last hypothesis (no scores of its own)
        dict(name="verify_stream", op="verify", streams=1, drafts=4, vocab=VOCAB, scores=False, greedy=False),
        # 64 streams with a draft model's scores
        dict(name="verify_batch", op="verify", streams=64, drafts=4, vocab=VOCAB, scores=True, greedy=False),
        # greedy decoding with long drafts
        dict(name="verify_greedy", op="verify", streams=16, drafts=10, vocab=VOCAB, scores=False, greedy=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "lora", "verify"])
    if op == "attn":
        rows = rng.choice([1, 1, 1, _log(rng, 1, 22)])
        dim = rng.choice([128, 128, 64])
        kv = rng.choice([1, 2, 4, 8, 16])
        group = rng.choice([1, 2, 3, 4, 5, 8])
        if kv * group > 32:
            group = 32 // kv
        return dict(op=op, seqs=_log(rng, 1, 64), rows=rows, prefix=_log(rng, 1, 8001), tail=rows + _log(rng, 1, 1000) - 1, ragged=rng.random() < 0.6,
                    heads=kv * group, kv_heads=kv, dim=dim)
    if op == "lora":
        K, N = rng.choice([QKV, O, DOWN, (64 * _log(rng, 4, 100), _log(rng, 48, 6144))])
        rows = _log(rng, 1, 320 if K > 8192 else 1408)
        rank = 8 * rng.choice([1, 2, 2, 3, 4, 8])
        return dict(op=op, rows=rows, K=K, N=N, rank=rank, adapters=_log(rng, 1, 64), spread=rng.choice(["runs", "mixed"]))
    greedy = rng.random() < 0.3
    return dict(op=op, streams=_log(rng, 1, 64), drafts=rng.randint(1, 4), vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]), scores=(not greedy) and rng.random() < 0.6,
                greedy=greedy)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case, seed):
    """(rows, tail keys) of every sequence: the same multiset for every seed, in another order."""
    B, T, L = case["seqs"], case["rows"], case["tail"]
    rows = [1 + (5 * b) % T if case["ragged"] else T for b in range(B)]
    # a tail holds the sequence's new rows at least; the longest is L
    tails = [rows[b] + (((B - 1 - b) * (L - rows[b])) // max(1, B - 1) if case["ragged"] else L - rows[b]) for b in range(B)]
    order = torch.randperm(B, generator=torch.Generator().manual_seed(seed)).tolist()
    return [rows[b] for b in order], [tails[b] for b in order]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    s = dict(case)
    if case["op"] == "attn":
        rows, tails = _lengths(case, seed)
        H, KV, D, P = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        cap = -(-case["tail"] // 64) * 64
        s["max_rows"] = max(rows)
        s["row_starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["tail_lens"] = torch.tensor(tails, dtype=torch.int32, device=DEV)
        s["q"] = normal(starts[-1], H, D)
        arena = normal(2, KV, -(-P // 64) * 64, D)  # slots behind the prefix are there, as in a cache, and not part of it
        s["k_prefix"], s["v_prefix"] = arena[0, :, :P], arena[1, :, :P]
        s["k_tail"], s["v_tail"] = normal(case["seqs"], KV, cap, D), normal(case["seqs"], KV, cap, D)
    elif case["op"] == "lora":
        M, K, N, r, A = (case[k] for k in ("rows", "K", "N", "rank", "adapters"))
        s["x"] = normal(M, K)
        W = normal(N, K, std=K ** -0.5)
        s["down"], s["up"] = normal(A, r, K, std=K ** -0.5), normal(A, N, r, std=0.3 * r ** -0.5)
        s["scales"] = torch.rand(A, generator=g, device=DEV) + 0.5
        # one row in sixteen runs without an adapter
        pick = torch.randint(0, 16 * A, (M,), generator=g, device=DEV)
        if case["spread"] == "runs":  # the rows of a stream are neighbours
            pick = pick[(torch.arange(M, device=DEV) // 22) * 22 % M]
        s["ids"] = torch.where(pick % 16 == 15, -1, pick // 16).to(torch.int32)
        if own:
            from infinisst_amd import engine
            s["packed"] = engine.op_pack_weight(W)
        else:
            s["W"] = W
    else:
        B, K, V = case["streams"], case["drafts"], case["vocab"]
        t = normal(B, K + 1, V, std=2.0, dtype=torch.float32)
        t.scatter_add_(2, torch.randint(0, V, (B, K + 1, 12), generator=g, device=DEV), normal(B, K + 1, 12, std=3.0, dtype=torch.float32) + 9.0)
        q = t[:, :K] + normal(B, K, V, std=0.5, dtype=torch.float32)
        s["target"] = t
        s["draft_scores"] = q if case["scores"] else None
        if case["scores"]:
            gumbel = -torch.log(-torch.log(torch.rand((B, K, V), generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7)))
            s["drafts"] = (q + gumbel).argmax(-1).to(torch.int32)
        else:  # mostly the model's own choice
            other = torch.randint(0, V, (B, K), generator=g, device=DEV)
            s["drafts"] = torch.where(torch.rand((B, K), generator=g, device=DEV) < 0.85, t[:, :K].argmax(-1), other).to(torch.int32)
        s["n_drafts"] = torch.randint(max(0, K - 1), K + 1, (B,), generator=g, device=DEV).to(torch.int32)
        s["uniforms"] = None if case["greedy"] else torch.rand((B, K + 1), generator=g, device=DEV, dtype=torch.float64)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        from infinisst_amd import engine
        if s["op"] == "attn":
            return engine.op_prefix_attention(s["q"], s["k_prefix"], s["v_prefix"], s["k_tail"], s["v_tail"], s["tail_lens"], s["row_starts"], s["max_rows"])
        if s["op"] == "lora":
            return engine.op_gemm_lora(s["x"], s["packed"], s["N"], s["down"], s["up"], s["scales"], s["ids"])
        return engine.op_verify_drafts(s["target"], s["drafts"], s["n_drafts"], s["draft_scores"], s["uniforms"])
    return {"attn": _attn, "lora": _lora, "verify": _verify}[s["op"]](s)


def _attn(s):
    R, H, D = s["q"].shape
    KV, B, T = s["kv_heads"], s["seqs"], s["max_rows"]
    G, L, scale = H // KV, s["k_tail"].shape[2], D ** -0.5
    starts, lens = s["row_starts"].long(), s["tail_lens"].long()
    n = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(B, device=DEV), n, output_size=R)
    at = torch.arange(R, device=DEV) - starts[seq]
    q = s["q"].float().view(R, KV, G, D)
    # scores against the prefix (every row, every key) and against the sequence's own keys (rows padded to T a sequence)
    sp = torch.matmul(q.permute(1, 0, 2, 3).reshape(KV, R * G, D), s["k_prefix"].float().transpose(1, 2)) * scale
    qt = torch.zeros(B, T, KV, G, D, device=DEV)
    qt[seq, at] = q
    st = torch.matmul(qt.permute(0, 2, 1, 3, 4).reshape(B, KV, T * G, D), s["k_tail"].float().transpose(2, 3)).view(B, KV, T, G, L) * scale
    sees = lens[:, None] - n[:, None] + torch.arange(T, device=DEV)[None] + 1  # row t of a sequence sees that many of its own keys
    hidden = torch.arange(L, device=DEV)[None, None] >= sees[:, :, None]
    st = st.masked_fill(hidden[:, None, :, None], -math.inf)
    st = st.permute(0, 2, 1, 3, 4)[seq, at]  # R, KV, G, L
    sp = sp.view(KV, R, G, -1).permute(1, 0, 2, 3)
    m = torch.maximum(sp.amax(-1), st.amax(-1))[..., None]
    m = torch.where(m == -math.inf, 0.0, m)
    ep, et = torch.exp(sp - m), torch.exp(st - m)
    total = ep.sum(-1) + et.sum(-1)
    o = torch.matmul(ep.permute(1, 0, 2, 3).reshape(KV, R * G, -1), s["v_prefix"].float()).view(KV, R, G, D).permute(1, 0, 2, 3)
    pt = torch.zeros(B, T, KV, G, L, device=DEV)
    pt[seq, at] = et
    v = torch.where((torch.arange(L, device=DEV)[None] < lens[:, None])[:, None, :, None], s["v_tail"].float(), 0.0)
    o = o + torch.matmul(pt.permute(0, 2, 1, 3, 4).reshape(B, KV, T * G, L), v).view(B, KV, T, G, D).permute(0, 2, 1, 3, 4)[seq, at]
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    return o.reshape(R, H, D).to(torch.bfloat16)


def _lora(s):
    x = s["x"].float()
    out = x @ s["W"].float().t()
    for r0 in range(0, x.shape[0], 256):  # (an adapter's matrices per row: in blocks of rows, for their size)
        ids = s["ids"][r0:r0 + 256].long()
        at = ids.clamp(min=0)
        t = torch.matmul(s["down"][at].float(), x[r0:r0 + 256, :, None])
        d = torch.matmul(s["up"][at].float(), t)[:, :, 0] * s["scales"][at][:, None]
        out[r0:r0 + 256] += torch.where((ids >= 0)[:, None], d, 0.0)
    return out.to(torch.bfloat16)


def _verify(s):
    # in 64 bits: a draw next to a border has to come out the same whatever the order of a sum
    t, n, x = s["target"].double(), s["n_drafts"].long(), s["drafts"].long()
    B, K, V = t.shape[0], t.shape[1] - 1, t.shape[2]
    b, index, steps = torch.arange(B, device=DEV), torch.arange(V, device=DEV), torch.arange(K, device=DEV)[None]
    if s["uniforms"] is None:
        best = torch.where(t == t.amax(-1, keepdim=True), index, V).amin(-1)
        accepted = ((best[:, :K] == x) & (steps < n[:, None])).long().cumprod(1).sum(1)
        pick = best[b, accepted]
    else:
        p = torch.exp(t - t.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        if s["draft_scores"] is None:
            q = torch.zeros_like(p[:, :K]).scatter_(2, x[:, :, None], 1.0)
        else:
            q = s["draft_scores"].double()
            q = torch.exp(q - q.amax(-1, keepdim=True))
            q = q / q.sum(-1, keepdim=True)
        u = s["uniforms"]
        px, qx = p[:, :K].gather(2, x[:, :, None])[..., 0], q.gather(2, x[:, :, None])[..., 0]
        accepted = ((u[:, :K] * qx < px) & (steps < n[:, None])).long().cumprod(1).sum(1)
        pr = p[b, accepted]
        w = (pr - q[b, accepted.clamp(max=K - 1)]).clamp(min=0.0)
        w = torch.where(((accepted < n) & (w.sum(-1) > 0))[:, None], w, pr)  # all accepted (or nothing left over): the model's own row
        run_ = w.cumsum(-1)
        hit = (run_ > u[:, K, None] * run_[:, -1:]) & (w > 0)
        pick = torch.where(hit, index, V).amin(-1)
        pick = torch.where(pick < V, pick, torch.where(w > 0, index, -1).amax(-1))
    out = torch.full((B, K + 1), -1, dtype=torch.int32, device=DEV)
    out[:, :K] = torch.where(steps < accepted[:, None], x, -1).to(torch.int32)
    out[b, accepted] = pick.to(torch.int32)
    return out, (accepted + 1).to(torch.int32)


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attn":
        rows, tails = _lengths(case, 0)
        H, KV, D, P = case["heads"], case["kv_heads"], case["dim"], case["prefix"]
        R = sum(rows)
        seen = sum(r * (t - r) + r * (r + 1) // 2 for r, t in zip(rows, tails))
        return {"bytes": 4 * R * H * D + 4 * KV * D * (P + sum(tails)) + 8 * len(rows) + 4, "flops": 4 * H * D * (R * P + seen)}
    if case["op"] == "lora":
        M, K, N, r = case["rows"], case["K"], case["N"], case["rank"]
        used = min(case["adapters"], -(-M // 22) if case["spread"] == "runs" else M)
        return {"bytes": 2 * (M * K + N * K + M * N + used * r * (K + N)) + 4 * M + 4 * case["adapters"], "flops": 2 * M * K * N + 2 * M * r * (K + N)}
    B, K, V = case["streams"], case["drafts"], case["vocab"]
    reads = B * (K + 1) + (B * K if case["scores"] else 0)
    return {"bytes": 4 * reads * V + (0 if case["greedy"] else 8 * B * (K + 1)) + 4 * B * (2 * K + 3), "flops": (1 if case["greedy"] else 4) * reads * V}


# ---------------------------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    if case["op"] == "attn":
        R, H, D = s["q"].shape
        KV = case["kv_heads"]
        out = torch.empty(R, H, D, dtype=torch.float64, device=DEV)
        starts, lens = s["row_starts"].tolist(), s["tail_lens"].tolist()
        kp, vp = s["k_prefix"].double(), s["v_prefix"].double()
        for b in range(case["seqs"]):
            n = starts[b + 1] - starts[b]
            k = torch.cat([kp, s["k_tail"][b, :, :lens[b]].double()], 1).repeat_interleave(H // KV, 0)  # H, keys, D
            v = torch.cat([vp, s["v_tail"][b, :, :lens[b]].double()], 1).repeat_interleave(H // KV, 0)
            sc = s["q"][starts[b]:starts[b + 1]].double().transpose(0, 1) @ k.transpose(1, 2) / math.sqrt(D)  # H, n, keys
            last = torch.arange(n, device=DEV) + k.shape[1] - n  # the newest key a row sees
            sc[:, torch.arange(k.shape[1], device=DEV)[None] > last[:, None]] = -math.inf
            out[starts[b]:starts[b + 1]] = (torch.softmax(sc, -1) @ v).transpose(0, 1)
        return out
    if case["op"] == "lora":
        x = s["x"].double()
        out = x @ s["W"].double().t()
        for a in range(case["adapters"]):
            rows = torch.nonzero(s["ids"] == a)[:, 0]
            if rows.numel():
                out[rows] += s["scales"][a].double() * (x[rows] @ s["down"][a].double().t() @ s["up"][a].double().t())
        return out
    import numpy as np
    B, K = case["streams"], case["drafts"]
    target, x, n = s["target"].cpu().numpy(), s["drafts"].tolist(), s["n_drafts"].tolist()
    scores = None if s["draft_scores"] is None else s["draft_scores"].cpu().numpy()
    u = None if s["uniforms"] is None else s["uniforms"].cpu().numpy()

    def softmax(row):
        e = np.exp(row.astype(np.float64) - float(row.max()))
        return e / e.sum()

    tokens, counts = torch.full((B, K + 1), -1, dtype=torch.int32), torch.empty(B, dtype=torch.int32)
    for b in range(B):
        i = 0
        while True:
            row = target[b, i]
            if u is None:
                pick = int(row.argmax())
                if i < n[b] and x[b][i] == pick:
                    tokens[b, i] = pick
                    i += 1
                    continue
            else:
                w = p = softmax(row)
                if i < n[b]:
                    q = softmax(scores[b, i]) if scores is not None else np.eye(1, p.size, x[b][i])[0]
                    if u[b, i] * q[x[b][i]] < p[x[b][i]]:
                        tokens[b, i] = x[b][i]
                        i += 1
                        continue
                    left = np.maximum(p - q, 0.0)
                    w = left if left.sum() > 0 else p
                total = np.cumsum(w)
                pick = min(int(np.searchsorted(total, u[b, K] * total[-1], side="right")), int(np.flatnonzero(w)[-1]))
            tokens[b, i] = pick
            counts[b] = i + 1
            break
    return tokens.to(DEV), counts.to(DEV)
