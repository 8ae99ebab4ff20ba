"""Shared-prefix attention, per-row low-rank adapters and draft verification on a real MI355X against 64-bit references.

Tolerances are worst-case bounds written down before the first run (u = half a step of a type, relative: bf16 2^-8, fp32 2^-24):
  attention  |o - ref| <= u_bf16 |ref| (the output's rounding) + (u_bf16 + 2^-12) A, A = softmax-weighted mean of |v|: the weights enter the value product as bf16 (u_bf16 each), and
             2^-12 covers the 32-bit part -- a score is D <= 128 products, scale * sum |q k| stays below 20 here, so its error is below 20 * 128 * 2^-24 < 2^-12.6, the exponential and the
             sums add a few 2^-24
  gemm_lora  |y - ref| <= u_bf16 |ref| + K u_fp32 sum |x w| + |s| (2 u_bf16^2 + (K + rank) u_fp32) sum_r (sum_k |x down|) |up|: fp32 sums of K (and rank) terms; the inner product enters the
             second product as a pair of bf16 numbers, whose residue is u_bf16^2
  verify     equal tokens and counts"""
import math

import numpy as np
import pytest
import torch

from infinisst_amd import engine as E

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, U_BF, U_F32 = torch.bfloat16, 2.0 ** -8, 2.0 ** -24


# ---------------------------------------------------------------------------------------------------------------- shared-prefix attention
def attn_inputs(seed, row_counts, lens, H, KV, D, P, cap, extra_rows=0, garbage=math.nan):
    """q, arenas and index tensors on the GPU; every slot behind the prefix and behind a sequence's own length holds `garbage`."""
    g = torch.Generator().manual_seed(seed)
    B, R = len(row_counts), sum(row_counts) + extra_rows
    q = torch.randn(R, H, D, generator=g).to(BF)
    kp, vp = (torch.full((KV, P + 5, D), garbage).to(BF) for _ in range(2))
    kp[:, :P], vp[:, :P] = torch.randn(KV, P, D, generator=g).to(BF), torch.randn(KV, P, D, generator=g).to(BF)
    kt, vt = (torch.full((B, KV, cap, D), garbage).to(BF) for _ in range(2))
    for b, l in enumerate(lens):
        l = min(max(l, 0), cap)
        kt[b, :, :l], vt[b, :, :l] = torch.randn(KV, l, D, generator=g).to(BF), torch.randn(KV, l, D, generator=g).to(BF)
    starts = torch.tensor([0] + np.cumsum(row_counts).tolist(), dtype=torch.int32)
    return q.to(DEV), kp.to(DEV)[:, :P], vp.to(DEV)[:, :P], kt.to(DEV), vt.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), starts.to(DEV)


def attn_ref(q, kp, vp, kt, vt, lens, starts, scale=None):
    """(o, A) in float64 on the CPU; NaN where no sequence owns the row."""
    q, kp, vp, kt, vt = (t.detach().cpu().double() for t in (q, kp, vp, kt, vt))
    R, H, D = q.shape
    KV, cap = kp.shape[0], kt.shape[2]
    G, scale = H // KV, D ** -0.5 if scale is None else scale
    o, A = torch.full((R, H, D), math.nan, dtype=torch.float64), torch.full((R, H, D), math.nan, dtype=torch.float64)
    starts, lens = starts.tolist(), lens.tolist()
    for b in range(len(lens)):
        n, l = starts[b + 1] - starts[b], min(max(lens[b], 0), cap)
        for t in range(n):
            see = min(max(l - n + t + 1, 0), l)
            k, v = torch.cat([kp, kt[b, :, :see]], 1), torch.cat([vp, vt[b, :, :see]], 1)
            r = starts[b] + t
            if k.shape[1] == 0:
                o[r] = A[r] = 0.0
                continue
            w = torch.softmax(torch.einsum("kgd,kjd->kgj", q[r].view(KV, G, D), k) * scale, -1)
            o[r], A[r] = (w @ v).reshape(H, D), (w @ v.abs()).reshape(H, D)
    return o, A


def attn_check(got, o, A, what=""):
    got = got.detach().cpu().double()
    live = ~torch.isnan(o)
    err, tol = (got - o).abs(), U_BF * o.abs() + (U_BF + 2.0 ** -12) * A + 1e-30
    bad = live & ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {int(live.sum())} off, worst {float((err / tol)[live].nan_to_num(1e9).max()):.3g} of the tolerance at {bad.nonzero()[0].tolist()}"


ATTN = {
    # name: (rows per sequence, own lengths, heads, key heads, D, prefix, capacity)
    "one_row_one_key": ([1], [1], 1, 1, 128, 0, 1),
    "one_prefix_key": ([1], [0], 4, 1, 128, 1, 8),
    "no_key_at_all": ([2, 1], [0, 0], 4, 2, 128, 0, 16),
    "first_rows_without_a_key": ([5, 3], [2, 3], 4, 2, 128, 0, 16),
    "own_longer_than_capacity": ([2, 2], [99, 7], 4, 4, 64, 33, 17),
    "negative_length": ([1, 1], [-3, 5], 4, 2, 128, 3, 8),
    "beams": ([1] * 4, [9, 9, 9, 9], 32, 8, 128, 1000, 64),
    "beams_no_prefix": ([1] * 4, [9, 64, 33, 31], 32, 8, 128, 0, 64),
    "ragged_rows": ([3, 0, 1, 22, 0, 7], [40, 9, 1, 100, 0, 7], 8, 2, 128, 129, 100),
    "drafts": ([5] * 12, [5, 6, 31, 32, 33, 63, 64, 65, 90, 128, 129, 200], 32, 8, 128, 257, 200),
    "many_rows": ([22, 40, 61], [22, 300, 61], 12, 4, 128, 511, 320),
    "long_prefix": ([2] * 3, [2, 5, 9], 4, 1, 128, 5003, 16),
    "many_columns": ([1] * 70, [1 + (7 * b) % 50 for b in range(70)], 8, 1, 128, 300, 64),
    "heads64": ([3, 1, 9], [70, 1, 9], 16, 16, 64, 200, 72),
    "heads64_grouped": ([33] * 5, [33, 64, 65, 100, 40], 10, 2, 64, 95, 100),
    "group_of_three": ([4, 17], [4, 80], 9, 3, 128, 77, 80),
    "group_of_seven": ([1, 2, 1], [50, 51, 52], 14, 2, 64, 1023, 64),
    "wide_group": ([1, 1], [5, 400], 48, 1, 128, 2049, 400),
    "one_long_sequence": ([150], [1200], 4, 4, 64, 64, 1200),
}


@pytest.mark.parametrize("name", list(ATTN))
def test_prefix_attention(name):
    rows, lens, H, KV, D, P, cap = ATTN[name]
    q, kp, vp, kt, vt, ln, st = attn_inputs(7, rows, lens, H, KV, D, P, cap)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    print(name, flush=True)
    got = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, max(rows))
    attn_check(got, o, A, name)
    # without the hint, with a wrong one, and again: the same bits whatever else runs
    for hint in (0, 1):
        attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, hint), o, A, f"{name}, max_rows {hint}")
    assert torch.equal(got, E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, max(rows)))
    if len(set(rows)) == 1:
        assert torch.equal(got, E.op_prefix_attention(q, kp, vp, kt, vt, ln))


@pytest.mark.parametrize("seed", range(24))
def test_prefix_attention_random_shapes(seed):
    rng = np.random.default_rng(100 + seed)
    B = int(rng.integers(1, 20))
    D, KV, G = int(rng.choice([64, 128])), int(rng.choice([1, 2, 5, 8])), int(rng.integers(1, 9))
    rows = [int(x) for x in rng.integers(0, int(rng.choice([2, 7, 40])), B)]
    rows[0] = max(rows[0], 1)
    lens = [int(r + rng.integers(0, int(rng.choice([2, 70, 300])))) for r in rows]
    P, scale = int(rng.choice([0, 1, 15, 31, 32, 33, 64, 100, 255, 700])), float(rng.choice([0.02, 0.125, 0.2]))
    q, kp, vp, kt, vt, ln, st = attn_inputs(seed, rows, lens, KV * G, KV, D, P, max(lens))
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st, scale)
    print(seed, rows, lens, KV, G, D, P, flush=True)
    attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, max(rows), scale=scale), o, A)


def test_prefix_attention_leaves_other_rows_alone():
    """Rows behind the last sequence (a padded batch), in front of the first and around a strided output keep their bytes."""
    q, kp, vp, kt, vt, ln, st = attn_inputs(3, [2, 3], [4, 9], 8, 2, 128, 50, 16, extra_rows=6)
    st = st + 2
    whole = torch.full((q.shape[0], 10, 160), 7.0, dtype=BF, device=DEV)
    out = whole[:, 1:9, 16:144]
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 3, out=out)
    attn_check(out, o, A)
    owned = ~torch.isnan(o[:, 0, 0])
    assert owned.tolist() == [False] * 2 + [True] * 5 + [False] * 4
    mask = torch.zeros(whole.shape, dtype=torch.bool)
    mask[owned, 1:9, 16:144] = True
    assert bool((whole.cpu()[~mask] == 7.0).all())


def test_prefix_attention_strided_views():
    """q inside fused q/k/v rows, key-major arenas ([slot][kv head]), the prefix inside a longer arena."""
    rows, lens, H, KV, D, P, cap = [3, 1, 8], [30, 1, 64], 8, 2, 128, 200, 64
    q, kp, vp, kt, vt, ln, st = attn_inputs(5, rows, lens, H, KV, D, P, cap)
    ref = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 8)
    fused = torch.randn(q.shape[0], (H + 2 * KV) * D, device=DEV).to(BF)
    fused[:, :H * D] = q.reshape(q.shape[0], -1)
    q2 = fused[:, :H * D].view(-1, H, D)
    turn = lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    kp2, vp2 = kp.transpose(0, 1).contiguous().transpose(0, 1), vp.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ref, E.op_prefix_attention(q2, kp2, vp2, turn(kt), turn(vt), ln, st, 8))
    # one arena for every sequence: broadcast keys
    one_k, one_v = kt[:1].expand(3, -1, -1, -1), vt[:1].expand(3, -1, -1, -1)
    ln2 = torch.tensor([30, 20, 10], dtype=torch.int32, device=DEV)
    o, A = attn_ref(q, kp, vp, one_k, one_v, ln2, st)
    attn_check(E.op_prefix_attention(q, kp, vp, one_k, one_v, ln2, st, 8), o, A)


def test_prefix_attention_masked_values_do_not_reach_a_row():
    """A newer row's own key and value hold NaN / inf: the rows that do not see it stay finite, the row that does shows it."""
    rows, lens, H, KV, D, P, cap = [4, 4], [20, 37], 4, 1, 128, 40, 64
    q, kp, vp, kt, vt, ln, st = attn_inputs(9, rows, lens, H, KV, D, P, cap)
    kt[0, :, 19], vt[0, :, 19] = math.nan, math.inf  # seen by the last row of sequence 0 only
    vt[1, :, 36, 3] = math.nan
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    got = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 4).cpu()
    ok = torch.ones(8, dtype=torch.bool)
    ok[[3, 7]] = False
    attn_check(got[ok], o[ok], A[ok])
    assert bool(torch.isnan(got[3]).all()) and bool(torch.isnan(got[7, :, 3]).all())
    keep = [d for d in range(D) if d != 3]
    attn_check(got[7][:, keep], o[7][:, keep], A[7][:, keep])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KV", [(4, 1), (2, 2)])
def test_prefix_attention_masked_values_among_many_columns(H, KV, D):
    """As above where a workgroup takes 128 columns: infinite and NaN values in neighbouring tiles that only the newest rows see, and in the last, partial tile of the prefix."""
    rows, lens, P, cap = [40, 70, 33], [100, 150, 33], 45, 160
    q, kp, vp, kt, vt, ln, st = attn_inputs(10, rows, lens, H, KV, D, P, cap)
    vt[0, 0, 95, 3], vt[0, 0, 97, 5], kt[0, 0, 99] = math.inf, math.nan, math.nan  # row t of sequence 0 sees the keys up to 60 + t
    vt[1, KV - 1, 120, 7], vt[1, :, 149], vt[1, 0, 127, 9], vt[1, 0, 128, 9] = math.nan, -math.inf, math.inf, math.inf  # ... of sequence 1 up to 80 + t
    vt[2, :, 1, 2], vt[2, :, 32, 60] = -math.inf, math.inf  # ... of sequence 2 up to t
    vp[0, 40, 11], vp[KV - 1, 44, 13] = math.inf, -math.inf
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    got = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 70).cpu().double()
    same = (torch.isnan(got) & torch.isnan(o)) | (got == o)
    fine = torch.isfinite(o)
    assert bool(same[~fine].all()), (~same & ~fine).nonzero()[:5]
    assert 0.5 < float(fine.double().mean()) < 1.0
    tol = U_BF * o.abs() + (U_BF + 2.0 ** -12) * A
    assert bool(((got - o).abs() <= tol)[fine].all()), (~((got - o).abs() <= tol) & fine).nonzero()[:5]


def test_prefix_attention_large_scores():
    """Scores in the thousands (one key takes everything) and scores that differ by less than a rounding."""
    q, kp, vp, kt, vt, ln, st = attn_inputs(11, [2, 2], [10, 70], 4, 2, 128, 100, 80)
    for mul in (30.0, 1e-3):
        qs = (q.float() * mul).to(BF)
        o, A = attn_ref(qs, kp, vp, kt, vt, ln, st)
        got = E.op_prefix_attention(qs, kp, vp, kt, vt, ln, st, 2).cpu().double()
        # scores 30 times larger: 30 times the error of a score (2^-12 above was for sum |q k| scale < 20)
        tol = U_BF * o.abs() + (U_BF + max(1.0, mul) * 2.0 ** -12) * A
        assert bool(((got - o).abs() <= tol).all())


@pytest.mark.parametrize("rows", [[1, 2], [40, 33]])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_prefix_attention_scores_of_two_to_the_24(rows, sign):
    """Scores of 2^24 and more, two apart, all of them exact in fp32 (8192 x 16384 + 16 n, times 1 / 8): their differences decide as between small scores."""
    H, KV, D, P, cap = 4, 2, 64, 300, 160
    q, kp, vp, kt, vt, ln, st = attn_inputs(25, rows, [r + 60 for r in rows], H, KV, D, P, cap)
    q.zero_()
    q[..., 0], q[..., 1] = 8192.0, 16.0
    kp[..., 0], kt[..., 0] = sign * 16384.0, sign * 16384.0
    kp[..., 1], kt[..., 1] = (torch.arange(P, device=DEV) * 7 % 5).to(BF), (torch.arange(cap, device=DEV) * 3 % 6).to(BF)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, max(rows)), o, A)


@pytest.mark.parametrize("rows,D", [([1, 2], 128), ([40, 33], 128), ([1] * 40, 64)])
@pytest.mark.parametrize("removed", [-math.inf, -3.3895313892515355e38])
def test_prefix_attention_scores_of_minus_infinity(rows, D, removed):
    """Keys whose scores are -inf (whole tiles of them, at the start of the prefix, of a span and of the own keys) leave the other keys' weights as they are, also where those are far below zero."""
    H, KV, P, cap = 4, 1, 700, 300
    lens = [n + 200 for n in rows]
    q, kp, vp, kt, vt, ln, st = attn_inputs(21, rows, lens, H, KV, D, P, cap)
    q[..., 0], q[..., 1] = 4.0, 64.0
    kp[..., 1], kt[:, :, :, 1] = -32.0, -32.0  # scores around -2048 / sqrt(D)
    kp[..., 0], kt[..., 0] = 0.0, 0.0
    kp[:, :170, 0] = kp[:, 300:420, 0] = kt[:, :, :130, 0] = removed
    kp[..., 0, 0] = removed
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    assert bool(torch.isfinite(o).all())
    got = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, max(rows)).cpu().double()
    # sum |q k| scale is 2048 / sqrt(D) here, not 20: its rounding, 2^-24 D of it, is below 2^-8
    tol = U_BF * o.abs() + (U_BF + 2.0 * 2.0 ** -24 * D * 2300 / math.sqrt(D)) * A
    assert bool(((got - o).abs() <= tol).all())


def test_prefix_attention_scores_that_grow():
    """Scores that rise by hundreds from the first keys on: every reference that a column starts with is far below its maximum."""
    rows, lens, H, KV, D, P, cap = [3, 30], [90, 200], 4, 2, 128, 900, 256
    q, kp, vp, kt, vt, ln, st = attn_inputs(23, rows, lens, H, KV, D, P, cap)
    q[..., 0] = 8.0
    kp[..., 0] = (torch.arange(P, device=DEV) * 0.5).to(BF)  # up to 8 * 450 / sqrt(128) = 318
    kt[..., 0] = (400 - torch.arange(cap, device=DEV)).to(BF)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    got = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 30).cpu().double()
    tol = U_BF * o.abs() + (U_BF + 2.0 * 2.0 ** -24 * D * 340) * A
    assert bool(((got - o).abs() <= tol).all())


def test_prefix_attention_offsets_past_32_bits():
    rows, lens, H, KV, D, P, cap = [1, 2], [40, 41], 4, 2, 128, 150, 48
    q, kp, vp, kt, vt, ln, st = attn_inputs(13, rows, lens, H, KV, D, P, cap)
    big = torch.zeros((1 << 31) + (1 << 28), dtype=BF, device=DEV)  # 4.8 GB
    far = lambda t, stride, at: big.as_strided(t.shape, stride, at)
    kp2, vp2 = far(kp, (D, (1 << 31) // P // 8 * 8, 1), 0), far(vp, (D, (1 << 31) // P // 8 * 8, 1), 512)
    kt2, vt2 = far(kt, (1 << 31, cap * D, D, 1), 1 << 20), far(vt, (1 << 31, cap * D, D, 1), (1 << 20) + (1 << 16))
    for dst, src in ((kp2, kp), (vp2, vp), (kt2, kt), (vt2, vt)):
        dst.copy_(src)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    attn_check(E.op_prefix_attention(q, kp2, vp2, kt2, vt2, ln, st, 2), o, A)


@pytest.mark.parametrize("R,H,KV,D", [(33, 1, 1, 128), (150, 4, 4, 64), (400, 8, 4, 128)])
def test_prefix_attention_every_number_of_tiles(R, H, KV, D):
    """Prefixes from one key to past four tiles of every remainder that matters, by columns of many rows at once (whatever spans the launch cuts them into)."""
    for P in list(range(1, 5)) + list(range(30, 36)) + list(range(62, 67)) + list(range(94, 100)) + [127, 128, 129, 160, 161, 191, 192, 193, 224, 225, 257, 289, 320, 353, 385]:
        q, kp, vp, kt, vt, ln, st = attn_inputs(P, [R], [0], H, KV, D, P, 8)
        print(R, P, flush=True)
        got = E.op_prefix_attention(q, kp, vp, kt[:, :, :0], vt[:, :, :0], ln, st, R).cpu().double()
        qd, k, v = (t.cpu().double() for t in (q, kp, vp))
        w = torch.softmax((qd.view(R, KV, H // KV, D).permute(1, 0, 2, 3).reshape(KV, -1, D) @ k.transpose(1, 2)) * D ** -0.5, -1)
        back = lambda x: x.view(KV, R, H // KV, D).permute(1, 0, 2, 3).reshape(R, H, D)
        attn_check(got, back(w @ v), back(w @ v.abs()), f"P {P}")


@pytest.mark.parametrize("rows", [9, 40, 70])
def test_prefix_attention_own_keys_of_every_length(rows):
    """Own keys of one sequence among others, from its rows alone to past four tiles: causal edges at every place of a tile."""
    for L in list(range(rows, rows + 36, 5)) + [95, 96, 97, 127, 128, 129, 150, 161, 193, 230, 260]:
        counts, lens = [1, rows, 2], [L // 2 + 1, max(L, rows), 3]
        q, kp, vp, kt, vt, ln, st = attn_inputs(L, counts, lens, 8, 2, 128, 37, 272)
        o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
        print(rows, L, flush=True)
        attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, rows), o, A, f"{rows} rows, {L} keys")


def test_prefix_attention_long_prefix_few_rows_and_wild_hints():
    q, kp, vp, kt, vt, ln, st = attn_inputs(31, [1, 2], [5, 60], 4, 1, 128, 60001, 64)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    for hint in (0, 2, 10 ** 9):
        attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, hint), o, A, f"max_rows {hint}")
    rows, lens = [150] + [1] * 30, [700] + [20] * 30  # one sequence far above the mean, which sizes the launch without a hint
    q, kp, vp, kt, vt, ln, st = attn_inputs(32, rows, lens, 4, 2, 64, 100, 700)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    for hint in (0, 1, 150):
        attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, hint), o, A, f"max_rows {hint}")


def test_prefix_attention_in_place_and_one_key_for_all():
    """The output in the place of the queries; a prefix whose keys are one row repeated (stride 0)."""
    rows, lens = [2, 40], [9, 50]
    q, kp, vp, kt, vt, ln, st = attn_inputs(33, rows, lens, 8, 2, 128, 90, 64)
    want = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 40)
    again = q.clone()
    assert E.op_prefix_attention(again, kp, vp, kt, vt, ln, st, 40, out=again) is again and torch.equal(again, want)
    one_k, one_v = kp[:, :1].expand(-1, 90, -1), vp[:, :1].expand(-1, 90, -1)
    o, A = attn_ref(q, one_k, one_v, kt, vt, ln, st)
    attn_check(E.op_prefix_attention(q, one_k, one_v, kt, vt, ln, st, 40), o, A)


def test_prefix_attention_head_major_output():
    """The output as a view of [heads][rows]: the same values, and nothing around them."""
    q, kp, vp, kt, vt, ln, st = attn_inputs(51, [2, 40], [9, 50], 8, 2, 128, 90, 64)
    want = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 40)
    whole = torch.full((8, 42, 144), 7.0, dtype=BF, device=DEV)
    out = whole[:, :, 8:136].transpose(0, 1)
    E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 40, out=out)
    assert torch.equal(out, want) and bool((whole[:, :, :8] == 7.0).all()) and bool((whole[:, :, 136:] == 7.0).all())


@pytest.mark.parametrize("R,L,P,H,KV,D", [(1500, 1500, 0, 4, 2, 128), (1100, 2300, 77, 3, 3, 64)])
def test_prefix_attention_whole_prompt_of_one_sequence(R, L, P, H, KV, D):
    """A prompt pass: every row of a long sequence at once, causal over its own keys, beside a sequence of one row."""
    q, kp, vp, kt, vt, ln, st = attn_inputs(41, [R, 1], [L, 5], H, KV, D, P, L)
    got = E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, R).cpu().double()
    qd = q.cpu().double()[:R].view(R, KV, H // KV, D).permute(1, 2, 0, 3)
    k, v = (torch.cat([x.cpu().double(), y[0, :, :L].cpu().double()], 1) for x, y in ((kp, kt), (vp, vt)))
    w = qd @ k[:, None].transpose(2, 3) * D ** -0.5
    w = torch.softmax(w.masked_fill(torch.arange(P + L)[None] > torch.arange(R)[:, None] + P + L - R, -math.inf), -1)
    back = lambda x: x.permute(2, 0, 1, 3).reshape(R, H, D)
    attn_check(got[:R], back(w @ v[:, None]), back(w @ v.abs()[:, None]))
    o, A = attn_ref(q[R:], kp, vp, kt[1:], vt[1:], ln[1:], torch.tensor([0, 1]))
    attn_check(got[R:], o, A)


@pytest.mark.parametrize("D", [64, 128])
def test_prefix_attention_long_own_keys(D):
    """One stream's row over tens of thousands of own keys (as many spans as the join takes), and a short one beside it."""
    q, kp, vp, kt, vt, ln, st = attn_inputs(43, [1, 3], [20011, 9], 4, 2, D, 0, 20011)
    o, A = attn_ref(q, kp, vp, kt, vt, ln, st)
    attn_check(E.op_prefix_attention(q, kp, vp, kt, vt, ln, st, 3), o, A)


def test_prefix_attention_without_any_slot():
    """No prefix and no room for own keys: every row of a sequence is zero, the others stay."""
    z = lambda *s: torch.empty(*s, dtype=BF, device=DEV)
    q, out = torch.randn(5, 4, 128, device=DEV).to(BF), torch.full((5, 4, 128), 3.0, dtype=BF, device=DEV)
    st = torch.tensor([1, 3, 4], dtype=torch.int32, device=DEV)
    E.op_prefix_attention(q, z(2, 0, 128), z(2, 0, 128), z(2, 2, 0, 128), z(2, 2, 0, 128), torch.tensor([7, 0], dtype=torch.int32, device=DEV), st, 2, out=out)
    assert out[:, 0, 0].tolist() == [3.0, 0.0, 0.0, 0.0, 3.0] and bool((out[1:4] == 0).all())


def test_prefix_attention_values_of_any_size():
    """Values up to 2^90 behind scores that rise by 14 in between (fp32 accumulators end at 2^128)."""
    rows, lens = [3, 30], [90, 60]
    q, kp, vp, kt, vt, ln, st = attn_inputs(34, rows, lens, 4, 2, 128, 300, 96)
    kp[:, 200:, 0], q[..., 0] = 20.0, 8.0
    for f in (2.0 ** 90, 2.0 ** -90):
        vp2, vt2 = vp * f, vt * f
        o, A = attn_ref(q, kp, vp2, kt, vt2, ln, st)
        got = E.op_prefix_attention(q, kp, vp2, kt, vt2, ln, st, 30).cpu().double()
        assert bool(((got - o).abs() <= U_BF * o.abs() + (U_BF + 2.0 ** -11) * A).all())  # (scores up to 34, not 20: 2^-12 becomes 2^-11)


@pytest.mark.parametrize("rows,lens,P", [([3, 30], [90, 60], 3000), ([1, 2], [40, 9], 6500)])
def test_prefix_attention_values_near_the_end_of_the_range(rows, lens, P):
    """Positive values up to 2^118 behind scores that rise by eight (eleven octaves) inside a span, too little for a new reference: the outputs end below 2^119, and no accumulator may pass 2^128."""
    q, kp, vp, kt, vt, ln, st = attn_inputs(35, rows, lens, 4, 2, 128, P, 96)
    at = torch.arange(P, device=DEV)
    q[..., 0], kt[..., 0] = 8.0, 0.0
    kp[..., 0] = torch.where((at // 32 % 4 > 1) if max(rows) > 8 else (at >= P // 2), 11.0, 0.0).to(BF)  # (two tiles low, two high; or the later steps of a wave)
    vp2, vt2 = vp.abs() * 2.0 ** 116, vt.abs() * 2.0 ** 116
    o, A = attn_ref(q, kp, vp2, kt, vt2, ln, st)
    got = E.op_prefix_attention(q, kp, vp2, kt, vt2, ln, st, max(rows)).cpu().double()
    assert bool(((got - o).abs() <= U_BF * o.abs() + (U_BF + 2.0 ** -11) * A).all())  # (scores up to 34, not 20: 2^-12 becomes 2^-11)


# ---------------------------------------------------------------------------------------------------------------- adapters
def lora_inputs(seed, M, N, K, rank, n, ids):
    g = torch.Generator().manual_seed(seed)
    x, W = torch.randn(M, K, generator=g).to(BF), (torch.randn(N, K, generator=g) * K ** -0.5).to(BF)
    down, up = (torch.randn(n, rank, K, generator=g) * K ** -0.5).to(BF), (torch.randn(n, N, rank, generator=g) * 0.5).to(BF)
    scales = torch.rand(n, generator=g) * 2 - 0.5
    return x, W, down, up, scales, torch.tensor(ids, dtype=torch.int32)


def lora_check(got, x, W, down, up, scales, ids, what=""):
    K, rank, n = x.shape[1], down.shape[1], down.shape[0]
    xd, Wd = x.double(), W.double()
    ref, mag = xd @ Wd.t(), K * U_F32 * (xd.abs() @ Wd.abs().t())
    for m, a in enumerate(ids.tolist()):
        if 0 <= a < n:
            s, d, u = float(scales[a]), down[a].double(), up[a].double()
            ref[m] += s * (u @ (d @ xd[m]))
            mag[m] += abs(s) * (2 * U_BF ** 2 + (K + rank) * U_F32) * (u.abs() @ (d.abs() @ xd[m].abs()))
    err, tol = (got.detach().cpu().double() - ref).abs(), U_BF * ref.abs() + mag + 1e-30
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max()):.3g} of the tolerance at {np.unravel_index(int((err / tol).argmax()), err.shape)}"


def lora_run(x, W, down, up, scales, ids, **kw):
    return E.op_gemm_lora(x.to(DEV), E.op_pack_weight(W.to(DEV)), W.shape[0], down.to(DEV), up.to(DEV), scales.to(DEV), ids.to(DEV), **kw)


@pytest.mark.parametrize("M", [1, 2, 5, 12, 13, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("N,K,rank", [(16, 32, 8), (1031, 256, 16), (272, 512, 24), (96, 1024, 64), (40, 96, 128)])
def test_gemm_lora(M, N, K, rank):
    n = 5
    ids = [(3 * m) % (n + 2) - 1 for m in range(M)]  # -1 and n: no adapter
    args = lora_inputs(M + N, M, N, K, rank, n, ids)
    print(M, N, K, rank, flush=True)
    got = lora_run(*args)
    lora_check(got, *args, what=f"M{M} N{N} K{K} r{rank}")
    assert torch.equal(got, lora_run(*args))


@pytest.mark.parametrize("M,N,K,rank,n,spread", [(64, 512, 4096, 16, 64, "each"), (200, 640, 2048, 32, 3, "runs"), (700, 272, 512, 16, 40, "mixed"), (330, 144, 8192, 40, 9, "mixed"),
                                                 (1, 6144, 4096, 16, 1, "runs"), (22, 4096, 1024, 8, 2, "runs"), (300, 64, 64, 8, 300, "each"), (257, 80, 160, 16, 1, "none")])
def test_gemm_lora_row_orders(M, N, K, rank, n, spread):
    rng = np.random.default_rng(M)
    ids = {"each": lambda: [m % n for m in range(M)], "runs": lambda: [(m // 22) % (n + 1) - 1 for m in range(M)],
           "mixed": lambda: rng.integers(-1, n, M).tolist(), "none": lambda: [-1] * M}[spread]()
    args = lora_inputs(M + K, M, N, K, rank, n, ids)
    print(M, N, K, rank, n, spread, flush=True)
    lora_check(lora_run(*args), *args, what=spread)


@pytest.mark.parametrize("M,N,K,rank", [(65, 2064, 4096, 16), (65, 2051, 4096, 16), (130, 2064, 4096, 32), (130, 2051, 4096, 16), (256, 2064, 4096, 64), (256, 2051, 4096, 16), (130, 600, 14336, 40)])
def test_gemm_lora_long_weights(M, N, K, rank):
    """65 to 256 rows of a weight of eight million entries and more (13 to 51 streams of five rows through a full-size projection): a base kernel of its own, whole and ragged columns."""
    n = 7
    rng = np.random.default_rng(M + N)
    args = lora_inputs(M + rank, M, N, K, rank, n, rng.integers(-1, n, M).tolist())
    print(M, N, K, rank, flush=True)
    got = lora_run(*args)
    lora_check(got, *args, what=f"M{M} N{N} K{K} r{rank}")
    assert torch.equal(got, lora_run(*args))


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 96, 128])
def test_gemm_lora_many_rows_of_every_rank(rank):
    """Enough rows and columns for the wide form of the adapter sum (1040 x 1031: 65 x 17 tiles), runs of rows and a changing adapter per row, a column tail, K past one slice."""
    M, N, n = 1040, 1031, 6
    for K, ids in ((96, [(m // 22) % (n + 1) - 1 for m in range(M)]), (1056, [(7 * m) % (n + 2) - 1 for m in range(M)])):
        args = lora_inputs(rank + K, M, N, K, rank, n, ids)
        print(rank, K, flush=True)
        lora_check(lora_run(*args), *args, what=f"rank {rank} K {K}")


def test_gemm_lora_adapters_do_not_mix():
    """An adapter of NaN / inf weights, a NaN scale and a NaN row reach their own rows only; wild ids mean no adapter."""
    M, N, K, rank, n = 40, 96, 256, 16, 4
    ids = [[0, 1, -1, 2, 3, 2 ** 31 - 1, -2 ** 31, n][m % 8] for m in range(M)]
    x, W, down, up, scales, ids = lora_inputs(1, M, N, K, rank, n, ids)
    clean = lora_run(x, W, down, up, scales, ids).cpu()
    down2, up2, scales2, x2 = down.clone(), up.clone(), scales.clone(), x.clone()
    down2[1, 3, 7], up2[2, 5], scales2[3], x2[0] = math.nan, math.inf, math.nan, math.nan
    got = lora_run(x2, W, down2, up2, scales2, ids).cpu()
    ill = (ids == 1) | (ids == 2) | (ids == 3)
    ill[0] = True
    assert torch.equal(got[~ill], clean[~ill])
    assert bool(torch.isnan(got[0]).all()) and bool(torch.isnan(got[ids == 1]).all()) and bool(torch.isnan(got[ids == 3]).all())
    hit = ids == 2
    assert not bool(torch.isfinite(got[hit][:, 5]).any()) and torch.equal(got[hit][:, 6:], clean[hit][:, 6:])


@pytest.mark.parametrize("M,N", [(40, 96), (1040, 1031)])
def test_gemm_lora_infinite_entries_have_the_sign_of_the_formula(M, N):
    """An infinite entry of `up` times an inner product that a bf16 number holds exactly, and one that it does not; zero times infinity is NaN; an inner product just below the end of fp32 stays finite."""
    K, rank = 256, 16
    g = torch.Generator().manual_seed(5)
    x, W = torch.zeros(M, K, dtype=BF), torch.zeros(N, K, dtype=BF)
    x[:, 0], x[:, 1] = torch.tensor([1.0, -2.0, 0.75, -96.0]).repeat(M)[:M].to(BF), torch.tensor([0.5, 0.0, -3.0]).repeat(M)[:M].to(BF)
    x[:, 2:60] = torch.randn(M, 58, generator=g).to(BF)
    x[:, 100], x[:, 101] = 3.3895313892515355e38, 2.0 ** 119
    down, up = torch.zeros(2, rank, K, dtype=BF), torch.zeros(2, N, rank, dtype=BF)
    down[1, 3, 0] = down[1, 0, 1] = down[1, 9, 100] = down[1, 9, 101] = 1.0
    down[1, 7, 2:60] = 0.25
    up[1, 5, 3], up[1, 9, 0], up[1, 13, 7], up[1, 17, 9] = math.inf, -math.inf, math.inf, 2.0 ** -90
    ids = torch.arange(M, dtype=torch.int32) % 3
    got = lora_run(x, W, down, up, torch.tensor([1.0, 1.0]), ids).double().cpu()
    rows = ids == 1
    xd = x.double()[rows]
    inner = xd[:, 2:60].sum(1)
    want = torch.zeros(int(rows.sum()), N, dtype=torch.float64)
    want[:, 5], want[:, 9], want[:, 13] = xd[:, 0] * math.inf, xd[:, 1] * -math.inf, inner * math.inf
    want[:, 17] = (xd[:, 100] + xd[:, 101]) * 2.0 ** -90  # (half way between the largest bf16 number and infinity)
    assert bool((got[~rows] == 0.0).all())
    ok = (got[rows] == want) | (torch.isnan(got[rows]) & torch.isnan(want)) | ((got[rows] - want).abs() <= U_BF * want.abs() + 2 * U_BF ** 2 * want.abs())
    assert bool(ok.all()), (~ok).nonzero()[:5]


def test_gemm_lora_strided():
    M, N, K, rank, n = 30, 144, 512, 16, 3
    x, W, down, up, scales, ids = lora_inputs(2, M, N, K, rank, n, [m % 4 - 1 for m in range(M)])
    wide = torch.full((M, 3 * K), 9.0, dtype=BF, device=DEV)
    wide[:, K:2 * K] = x.to(DEV)
    out = torch.full((M, N + 24), 5.0, dtype=BF, device=DEV)
    ref = lora_run(x, W, down, up, scales, ids)
    got = E.op_gemm_lora(wide[:, K:2 * K], E.op_pack_weight(W.to(DEV)), N, down.to(DEV), up.to(DEV), scales.to(DEV), ids.to(DEV), out=out[:, 8:8 + N])
    assert torch.equal(got, ref) and bool((out[:, :8] == 5.0).all()) and bool((out[:, 8 + N:] == 5.0).all())


def test_gemm_lora_millions_of_rows():
    """More rows than 65535 workgroups of the kernel without K slices take (64 rows each), at the smallest depth and width; 1009 rows repeated."""
    M, N, K, rank, n, period = 64 * 65535 + 77, 16, 32, 8, 3, 1009
    x, W, down, up, scales, ids = lora_inputs(7, period, N, K, rank, n, [m % 4 - 1 for m in range(period)])
    many = torch.arange(M, device=DEV) % period
    got = E.op_gemm_lora(x.to(DEV)[many], E.op_pack_weight(W.to(DEV)), N, down.to(DEV), up.to(DEV), scales.to(DEV), ids.to(DEV)[many])
    first = got[:period]
    lora_check(first, x, W, down, up, scales, ids)
    assert torch.equal(got, first[many])  # (a row's sums do not depend on where it stands)


def test_gemm_lora_in_place():
    M, K, rank, n = 70, 256, 16, 4
    x, W, down, up, scales, ids = lora_inputs(3, M, K, K, rank, n, [m % 5 - 1 for m in range(M)])
    want, xd = lora_run(x, W, down, up, scales, ids), x.to(DEV)
    E.op_gemm_lora(xd, E.op_pack_weight(W.to(DEV)), K, down.to(DEV), up.to(DEV), scales.to(DEV), ids.to(DEV), out=xd)
    assert torch.equal(xd, want)


# ---------------------------------------------------------------------------------------------------------------- drafts
def softmax64(row):
    e = np.exp(row.astype(np.float64) - float(row.max()))
    return e / e.sum()


def verify_ref(target, drafts, n_drafts, draft_scores, uniforms):
    B, K, V = target.shape[0], target.shape[1] - 1, target.shape[2]
    tokens, counts = np.full((B, K + 1), -1, np.int32), np.full(B, -1, np.int32)
    has = lambda row: not (np.isnan(row).any() or (row == np.inf).any() or not np.isfinite(row).any())
    for b in range(B):
        n, out, i = K if n_drafts is None else int(n_drafts[b]), [], 0
        if not 0 <= n <= K or (uniforms is not None and not 0 <= uniforms[b, K] < 1):
            continue
        while True:
            row = target[b, i]
            if not has(row):
                out = None
                break
            if i < n:
                x = int(drafts[b, i])
                if not 0 <= x < V or (draft_scores is not None and not has(draft_scores[b, i])) or (uniforms is not None and not 0 <= uniforms[b, i] < 1):
                    out = None
                    break
                if uniforms is None:
                    ok = x == int(row.argmax())
                else:
                    p = softmax64(row)
                    q = softmax64(draft_scores[b, i]) if draft_scores is not None else (np.arange(V) == x).astype(np.float64)
                    ok = uniforms[b, i] * q[x] < p[x]
                if ok:
                    out.append(x)
                    i += 1
                    continue
            if uniforms is None:
                out.append(int(row.argmax()))
                break
            w = softmax64(row)
            if i < n:
                left = np.maximum(p - q, 0.0)
                w = left if left.sum() > 0 else w
            cum = np.cumsum(w)
            live = np.flatnonzero(w > 0)
            hit = live[cum[live] > uniforms[b, K] * cum[-1]]
            out.append(int(hit[0]) if hit.size else int(live[-1]))
            break
        if out is not None:
            tokens[b, :len(out)], counts[b] = out, len(out)
    return tokens, counts


def verify_inputs(seed, B, K, V, spread=2.0):
    rng = np.random.default_rng(seed)
    t = (rng.standard_normal((B, K + 1, V)) * spread).astype(np.float32)
    q = (t[:, :K] + rng.standard_normal((B, K, V)) * 0.7).astype(np.float32)
    drafts = (q + rng.gumbel(size=q.shape)).argmax(-1).astype(np.int32)
    n = rng.integers(0, K + 1, B).astype(np.int32)
    return t, drafts, n, q, rng.random((B, K + 1))


def verify_run(t, drafts, n, q, u):
    up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    tokens, counts = E.op_verify_drafts(up(t), up(drafts), up(n), up(q), up(u))
    return tokens.cpu().numpy(), counts.cpu().numpy()


def verify_same(args):
    got, want = verify_run(*args), verify_ref(*args)
    assert np.array_equal(got[1], want[1]), (got[1], want[1])
    assert np.array_equal(got[0], want[0]), np.argwhere(got[0] != want[0])[:5]


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 2), (3, 2, 5), (2, 0, 300), (17, 3, 255), (5, 8, 257), (4, 4, 1031), (3, 5, 8193), (2, 4, 128263), (300, 1, 70)])
@pytest.mark.parametrize("kind", ["scores", "bare", "greedy"])
def test_verify_drafts(B, K, V, kind):
    for seed in range(3):
        t, drafts, n, q, u = verify_inputs(1000 * seed + V, B, K, V)
        if kind != "scores" and K:  # drafts that a target without noise would often accept
            drafts = np.where(np.random.default_rng(seed).random((B, K)) < 0.7, t[:, :K].argmax(-1), drafts).astype(np.int32)
        verify_same((t, drafts, None if seed == 2 else n, q if kind == "scores" and K else None, None if kind == "greedy" else u))


def long_drafts(seed, B, K, V, stops, kind):
    """Inputs whose stream b accepts stops[b][1] of stops[b][0] drafts: target and draft agree on the drafted token but at the refusal."""
    t, drafts, n, q, u = verify_inputs(seed, B, K, V)
    at = np.arange(K)
    for b, (live, accepted) in enumerate(stops):
        n[b] = live
        t[b, at, drafts[b]] += 30.0
        q[b, at, drafts[b]] += 28.0
        if accepted < live:
            t[b, accepted, drafts[b, accepted]] -= 60.0
    return t, drafts, n, q if kind == "scores" else None, None if kind == "greedy" else u


@pytest.mark.parametrize("kind", ["scores", "bare", "greedy"])
def test_verify_drafts_more_than_32(kind):
    K = 70
    stops = [(70, a) for a in (0, 1, 31, 32, 33, 63, 64, 65, 69, 70)] + [(n, n) for n in (0, 31, 32, 33, 64, 65)] + [(33, 32), (65, 64), (32, 31)]
    args = long_drafts(3, len(stops), K, 300, stops, kind)
    assert verify_ref(*args)[1].tolist() == [a + 1 for _, a in stops]
    verify_same(args)


@pytest.mark.parametrize("V", [131073, 151936, 262145, 300001])
@pytest.mark.parametrize("kind", ["scores", "bare", "greedy"])
def test_verify_drafts_large_vocabularies(V, kind):
    """More than 32 and more than 64 slices of 4096 scores; draws at both ends and past slice 64, drafts in the last slice, whole slices of removed entries."""
    B, K = 6, 2
    t, drafts, n, q, u = verify_inputs(V, B, K, V)
    n[:] = K
    drafts[3:, 0] = V - 1 - np.arange(3)
    u[:, K] = [0.0, 0.5, 0.93, 0.9999, 1.0 - 2.0 ** -53, 0.97]
    u[:, 0] = np.where(np.arange(B) % 2, 0.999999, u[:, 0])  # (mostly refused)
    t[2, :, 4096 * 3:4096 * 30] = -np.inf
    t[5, :, :V - 40] = -np.inf
    drafts[5] = V - 7
    if kind == "greedy":
        drafts[:] = t[:, :K].argmax(-1)
        drafts[1, 1] += -1 if drafts[1, 1] else 1
        t[4, 1, V - 1] = t[4, 1, 5] = 60.0
        drafts[4, 1] = 5
    verify_same((t, drafts, n, q if kind == "scores" else None, None if kind == "greedy" else u))


def test_verify_drafts_ties_and_removed_entries():
    """Greedy ties go to the lowest index; -inf entries are never drawn nor accepted; identical rows accept everything and their draw falls back to the row."""
    B, K, V = 6, 3, 5000
    t, drafts, n, q, u = verify_inputs(4, B, K, V)
    t[:, :, 7], t[:, :, 4321] = 50.0, 50.0
    drafts[:3], drafts[3:] = 7, 4321
    verify_same((t, drafts, n, None, None))
    t, drafts, n, q, u = verify_inputs(5, B, K, V)
    t[:, :, ::2] = -np.inf
    q[:, :, 1::3] = -np.inf
    verify_same((t, drafts, None, q, u))
    verify_same((t, drafts, None, None, u))
    t[:, :, :] = -np.inf
    t[:, :, 4999] = -3.0
    verify_same((t, np.full_like(drafts, 4999), None, None, u))
    t, drafts, n, q, u = verify_inputs(6, B, K, V)
    verify_same((t, drafts, None, t[:, :K].copy(), u))
    for edge in (0.0, 1.0 - 2.0 ** -53):
        verify_same((t, drafts, None, q, np.full_like(u, edge)))


def test_verify_drafts_bad_rows_name_their_stream_only():
    B, K, V = 9, 3, 700
    t, drafts, n, q, u = verify_inputs(8, B, K, V)
    n[:] = K
    t[0, 0, 5], t[1, 0, 699], t[2, 0, :] = np.nan, np.inf, -np.inf
    q[3, 0, 1] = np.nan
    drafts[4, 0], drafts[5, 0] = V, -1
    n[6], n[7] = K + 1, -1
    u[8, K] = 1.0
    want = verify_ref(t, drafts, n, q, u)
    assert (want[1] == -1).sum() == 9
    verify_same((t, drafts, n, q, u))
    # a bad row behind the first refusal does not matter
    t, drafts, n, q, u = verify_inputs(9, 4, K, V)
    n[:], t[:, 0, 0] = K, 60.0
    drafts[:, 0] = 1
    t[:, 2:] = np.nan
    q[:, 1:] = np.nan
    drafts[:, 1:] = 10 ** 9
    assert (verify_ref(t, drafts, n, q, u)[1] == 1).all()
    verify_same((t, drafts, n, q, u))


def test_verify_drafts_rows_behind_the_drafts_do_not_matter():
    B, K, V = 8, 5, 4500
    for kind in ("scores", "bare", "greedy"):
        t, drafts, n, q, u = verify_inputs(12, B, K, V)
        n[:] = np.arange(B) % (K + 1)
        drafts = np.where(np.random.default_rng(3).random((B, K)) < 0.8, t[:, :K].argmax(-1), drafts).astype(np.int32)
        if kind == "scores":  # a draft that is sure of its token, as the target is: accepted mostly
            t[np.arange(B)[:, None], np.arange(K), drafts] += 20.0
            q[np.arange(B)[:, None], np.arange(K), drafts] += 18.0
        for b in range(B):
            t[b, n[b] + 1:], q[b, n[b]:], drafts[b, n[b]:] = np.nan, np.inf, -5
        want = verify_ref(t, drafts, n, q if kind == "scores" else None, None if kind == "greedy" else u)
        assert (want[1] > 0).all() and (want[1] == n + 1).sum() >= 2
        verify_same((t, drafts, n, q if kind == "scores" else None, None if kind == "greedy" else u))


@pytest.mark.parametrize("B,V", [(64, 50), (16, 5000)])
def test_verify_drafts_compare_in_64_bits(B, V):
    """A draft without scores is accepted at a uniform 2^-46 (relative) below its probability and refused 2^-46 above it.  The probability's own error is below half of that: an exponential 1.3e-15
    (its polynomial 4.3e-16, the reduced argument 2.4e-17 |k| with |k| <= 36), up to 40 additions and products of a sum 4.5e-15, 1.3e-15 for its terms, the quotient 1.1e-16."""
    from decimal import Decimal, localcontext
    rng = np.random.default_rng(V)
    t = (rng.standard_normal((B, 2, V)) * 2.0).astype(np.float32)
    drafts = rng.integers(0, V, (B, 1)).astype(np.int32)
    drafts[: B // 2, 0] = t[: B // 2, 0].argmax(-1)
    p = []
    with localcontext() as ctx:
        ctx.prec = 40
        for b in range(B):
            e = [(Decimal(float(s)) - Decimal(float(t[b, 0].max()))).exp() for s in t[b, 0]]
            p.append(e[drafts[b, 0]] / sum(e))
        u = np.array([[[float(pb * (1 + side * Decimal(2) ** -46)), 0.5] for pb in p] for side in (-1, 1)])
    below, above = verify_run(t, drafts, None, None, u[0])[1], verify_run(t, drafts, None, None, u[1])[1]
    assert (below == 2).all() and (above == 1).all(), (int((below != 2).sum()), int((above != 1).sum()))


def test_verify_drafts_strided_scores():
    t, drafts, n, q, u = verify_inputs(10, 3, 2, 1031)
    wide = torch.zeros(3, 4, 1100, device=DEV)
    wide[:, :3, 5:1036] = torch.from_numpy(t).to(DEV)
    wq = torch.zeros(2, 3, 1035, device=DEV)
    wq[:, :, :1031] = torch.from_numpy(q).to(DEV).transpose(0, 1)
    up = lambda a: torch.from_numpy(a).to(DEV)
    tokens, counts = E.op_verify_drafts(wide[:, :3, 5:1036], up(drafts), up(n), wq.transpose(0, 1)[:, :, :1031], up(u))
    want = verify_ref(t, drafts, n, q, u)
    assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(counts.cpu().numpy(), want[1])


def test_verify_drafts_follow_the_target_distribution():
    """Whatever the draft proposes, the first token is distributed as the target's softmax: 40 000 independent streams over 6 tokens (each expected count within 5 sigma)."""
    B, V = 40000, 6
    rng = np.random.default_rng(1)
    p, q = np.log(np.array([.3, .05, .2, .15, .1, .2])), np.log(np.array([.1, .4, .1, .1, .2, .1]))
    drafts = rng.choice(V, size=(B, 1), p=np.exp(q)).astype(np.int32)
    t = np.broadcast_to(p.astype(np.float32), (B, 2, V))
    tokens, counts = verify_run(t, drafts, None, np.broadcast_to(q.astype(np.float32), (B, 1, V)), rng.random((B, 2)))
    assert set(np.unique(counts)) == {1, 2}
    seen = np.bincount(tokens[:, 0], minlength=V)
    assert (np.abs(seen - B * np.exp(p)) < 5 * np.sqrt(B * np.exp(p) * (1 - np.exp(p)))).all(), seen


# ---------------------------------------------------------------------------------------------------------------- together
def step_state(seed, B=6, K=3, KV=2, G=4, D=128, dim=256, V=1031, P=90, cap=64, rank=16, n=3):
    g = torch.Generator().manual_seed(seed)
    T, H = K + 1, KV * G
    normal = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(BF).to(DEV)
    w = {"qkv": ((H + 2 * KV) * D, dim), "o": (dim, H * D), "head": (V, dim)}
    s = dict(B=B, K=K, T=T, H=H, KV=KV, D=D, V=V, x=normal(B * T, dim), kp=normal(KV, P, D), vp=normal(KV, P, D), kt=normal(B, KV, cap, D), vt=normal(B, KV, cap, D),
             lens=torch.tensor([T + (11 * b) % 50 for b in range(B)], dtype=torch.int32, device=DEV), scales=torch.tensor([0.5, 1.0, 2.0], device=DEV),
             ids=torch.tensor([b % (n + 1) - 1 for b in range(B) for _ in range(T)], dtype=torch.int32, device=DEV), drafts=torch.zeros(B, K, dtype=torch.int32, device=DEV),
             uniforms=torch.rand(B, K + 1, generator=g, dtype=torch.float64).to(DEV))
    for name, (N, k) in w.items():
        s["w_" + name] = normal(N, k, std=k ** -0.5)
        s["p_" + name] = E.op_pack_weight(s["w_" + name])
        s["d_" + name], s["u_" + name] = normal(n, rank, k, std=k ** -0.5), normal(n, N, rank, std=0.2)
    return s


def step(s, uniforms=None):
    """One pass over B streams x (K + 1) rows: adapted q/k/v, the new keys into the tails, attention, adapted output projection, scores, verification."""
    B, T, H, KV, D = s["B"], s["T"], s["H"], s["KV"], s["D"]
    lora = lambda x, name: E.op_gemm_lora(x, s["p_" + name], s["w_" + name].shape[0], s["d_" + name], s["u_" + name], s["scales"], s["ids"])
    qkv = lora(s["x"], "qkv").view(B, T, H + 2 * KV, D)
    at = (s["lens"].long()[:, None] - T + torch.arange(T, device=DEV))
    b = torch.arange(B, device=DEV)[:, None]
    s["kt"].transpose(1, 2)[b, at], s["vt"].transpose(1, 2)[b, at] = qkv[:, :, H:H + KV], qkv[:, :, H + KV:]
    ctx = E.op_prefix_attention(qkv.view(B * T, -1, D)[:, :H], s["kp"], s["vp"], s["kt"], s["vt"], s["lens"])
    h = lora(ctx.view(B * T, H * D), "o")
    scores = E.op_gemm(h, s["p_head"], s["V"], "f32").view(B, T, s["V"])
    return (qkv, ctx, h, scores) + E.op_verify_drafts(scores, s["drafts"], None, None, uniforms)


def test_decode_step_of_drafted_streams():
    s = step_state(0)
    first = step(s)
    s["drafts"].copy_(first[3][:, :s["K"]].argmax(-1).to(torch.int32))  # drafts that greedy verification accepts
    s["drafts"][1, 1] = 5
    for uniforms in (None, s["uniforms"]):
        qkv, ctx, h, scores, tokens, counts = step(s, uniforms)
        cpu = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
        lora_check(qkv.reshape(-1, s["w_qkv"].shape[0]), cpu["x"], cpu["w_qkv"], cpu["d_qkv"], cpu["u_qkv"], cpu["scales"], cpu["ids"])
        starts = torch.arange(0, s["B"] * s["T"] + 1, s["T"])
        o, A = attn_ref(qkv.view(-1, s["H"] + 2 * s["KV"], s["D"])[:, :s["H"]], s["kp"], s["vp"], s["kt"], s["vt"], s["lens"], starts)
        attn_check(ctx, o, A)
        lora_check(h, ctx.view(s["B"] * s["T"], -1).cpu(), cpu["w_o"], cpu["d_o"], cpu["u_o"], cpu["scales"], cpu["ids"])
        want = verify_ref(scores.cpu().numpy(), cpu["drafts"].numpy(), None, None, None if uniforms is None else uniforms.cpu().numpy())
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(counts.cpu().numpy(), want[1])
        if uniforms is None:
            assert counts.tolist() == [4, 2, 4, 4, 4, 4]


def test_decode_step_captured_and_replayed():
    """The step as a graph: new inputs through the captured buffers, several replays with eager work between them, every replay against the eager result; two graphs at once."""
    s, other = step_state(1), step_state(2, B=5, P=33)
    side = torch.cuda.Stream()
    graphs = []
    for st in (s, other):
        with torch.cuda.stream(side):
            step(st, st["uniforms"])
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(st, st["uniforms"])
        graphs.append((g, out, st))
    for r in range(4):
        for g, out, st in graphs:
            st["x"].copy_(torch.randn(st["x"].shape, generator=torch.Generator().manual_seed(50 + r)).to(BF))
            st["lens"].copy_(torch.tensor([st["T"] + (13 * b + 7 * r) % 55 for b in range(st["B"])], dtype=torch.int32))
        torch.cuda.synchronize()
        for g, out, st in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out, st in graphs:
            for a, b in zip(out, step(st, st["uniforms"])):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    states = [step_state(s) for s in (3, 4)]
    want = [step(s, s["uniforms"]) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = []
    for s, st in zip(states, streams):
        with torch.cuda.stream(st):
            got.append([step(s, s["uniforms"]) for _ in range(5)])
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, run))


def test_empty_batches():
    z = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device=DEV)
    assert E.op_prefix_attention(z(0, 4, 128), z(2, 3, 128), z(2, 3, 128), z(0, 2, 8, 128), z(0, 2, 8, 128), z(0, dt=torch.int32)).shape == (0, 4, 128)
    W = torch.ones(16, 32, dtype=BF, device=DEV)
    assert E.op_gemm_lora(z(0, 32), E.op_pack_weight(W), 16, z(1, 8, 32), z(1, 16, 8), z(1, dt=torch.float32), z(0, dt=torch.int32)).shape == (0, 16)
    tokens, counts = E.op_verify_drafts(z(0, 3, 10, dt=torch.float32), z(0, 2, dt=torch.int32))
    assert tokens.shape == (0, 3) and counts.shape == (0,)
