"""What the entry points of shared-prefix attention, per-row adapters and draft verification refuse, on the CPU: the C ABI answers before it launches anything, the Python
functions before they call it."""
import ctypes as C

import pytest
import torch

from infinisst_amd import engine as E

FAKE = 1 << 20  # a 16-byte aligned address nothing looks at


@pytest.fixture
def lib(built_library):
    return E.load_library()


def attn(**kw):
    a = E._PrefixAttn(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE)
    for n, v in dict(q_row=512, q_head=128, out_row=512, out_head=128, kp_head=12800, kp_key=128, vp_head=12800, vp_key=128, kt_seq=2048, kt_head=1024, kt_key=128, vt_seq=2048,
                     vt_head=1024, vt_key=128, rows=3, seqs=2, max_rows=2, heads=4, kv_heads=2, head_dim=128, prefix_len=100, tail_cap=8, scale=0.1).items():
        setattr(a, n, v)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(seqs=0), dict(seqs=-1), dict(max_rows=-1), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(head_dim=96), dict(prefix_len=-1),
                                 dict(tail_cap=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=None),
                                 dict(tail_lens=None), dict(k_prefix=None), dict(v_tail=None), dict(q=FAKE + 2), dict(out=FAKE + 8), dict(v_prefix=FAKE + 4), dict(q_row=516),
                                 dict(kp_key=129), dict(vt_seq=2044), dict(out_head=64), dict(out_row=256), dict(row_starts=None), dict(rows=1 << 30)])
def test_prefix_attention_refuses(lib, bad):
    a = attn(**bad)
    assert lib.isst_op_prefix_attention_workspace(C.byref(a)) == -1
    assert lib.isst_op_prefix_attention(C.byref(a), FAKE, 1 << 40, None) == -1


def test_prefix_attention_size_limits(lib):
    """rows * heads <= 2^26, seqs * kv_heads <= 2^22, heads <= 2^15, a key's stride <= 2^24: the limits themselves are taken, one more is not."""
    ws = lambda **kw: lib.isst_op_prefix_attention_workspace(C.byref(attn(**kw)))
    assert ws(rows=1 << 24) >= (1 << 26) * (128 * 4 + 8) and ws(rows=(1 << 24) + 1) == -1
    assert ws(seqs=1 << 21, max_rows=1 << 30) > 0 and ws(seqs=(1 << 21) + 1) == -1
    assert ws(heads=1 << 15, kv_heads=1, q_row=1 << 22, out_row=1 << 22) > 0 and ws(heads=1 << 16, kv_heads=1, q_row=1 << 23, out_row=1 << 23) == -1
    for key in ("kp_key", "vp_key", "kt_key", "vt_key"):
        assert ws(**{key: 1 << 24}) > 0 and ws(**{key: (1 << 24) + 8}) == -1 and ws(**{key: -8}) == -1


def test_prefix_attention_output_orders(lib):
    """Outputs of a row together or of a head together, never overlapping (3 rows, 4 heads of 128)."""
    ws = lambda row, head, **kw: lib.isst_op_prefix_attention_workspace(C.byref(attn(out_row=row, out_head=head, **kw)))
    assert ws(512, 128) > 0 and ws(128, 384) > 0 and ws(136, 400) > 0 and ws(1 << 40, 1 << 20) > 0 and ws(1 << 20, 1 << 40) > 0
    for row, head in ((504, 128), (128, 376), (120, 400), (512, 120), (128, 128), (0, 384), (-128, 512), (512, -128)):
        assert ws(row, head) == -1, (row, head)
    assert ws(0, 128, rows=1, seqs=1) > 0 and ws(128, 0, heads=1, kv_heads=1) > 0


def test_prefix_attention_workspace(lib):
    assert lib.isst_op_prefix_attention(None, None, 0, None) == -1 and lib.isst_op_prefix_attention_workspace(None) == -1
    a = attn()
    need = lib.isst_op_prefix_attention_workspace(C.byref(a))
    assert need >= 0
    if need:
        assert lib.isst_op_prefix_attention(C.byref(a), FAKE, need - 1, None) == -4
        assert lib.isst_op_prefix_attention(C.byref(a), None, need, None) == -1
        assert lib.isst_op_prefix_attention(C.byref(a), FAKE + 4, need, None) == -1
    none = attn(rows=0, seqs=0)
    assert lib.isst_op_prefix_attention_workspace(C.byref(none)) == 0 and lib.isst_op_prefix_attention(C.byref(none), None, 0, None) == 0


def lora(lib, **kw):
    v = dict(A=FAKE, lda=256, packed=FAKE, down=FAKE, up=FAKE, scales=FAKE, ids=FAKE, n=3, rank=16, out=FAKE, ldo=64, M=5, N=64, K=256, ws=FAKE, bytes=1 << 40)
    v.update(kw)
    return lib.isst_op_gemm_lora(v["A"], v["lda"], v["packed"], v["down"], v["up"], v["scales"], v["ids"], v["n"], v["rank"], v["out"], v["ldo"], v["M"], v["N"], v["K"], v["ws"],
                                 v["bytes"], None)


@pytest.mark.parametrize("bad", [dict(A=None), dict(packed=None), dict(down=None), dict(up=None), dict(scales=None), dict(ids=None), dict(out=None), dict(ws=None), dict(A=FAKE + 2),
                                 dict(packed=FAKE + 8), dict(down=FAKE + 8), dict(up=FAKE + 2), dict(ws=FAKE + 4), dict(n=0), dict(rank=0), dict(rank=12), dict(rank=136), dict(K=250),
                                 dict(K=0), dict(N=0), dict(M=-1), dict(lda=248), dict(lda=260), dict(ldo=63), dict(M=1 << 30), dict(lda=1 << 30)])
def test_gemm_lora_refuses(lib, bad):
    assert lora(lib, **bad) == -1


def test_gemm_lora_workspace(lib):
    need = lib.isst_op_gemm_lora_workspace(5, 64, 256, 16, 3)
    assert need >= 4 * 5 * (64 + 16)
    assert lora(lib, bytes=need - 1) == -4 and lora(lib, M=0) == 0
    assert lib.isst_op_gemm_lora_workspace(5, 64, 250, 16, 3) == -1


def verify(lib, **kw):
    v = dict(t=FAKE, ts=300, tr=100, q=FAKE, qs=200, qr=100, drafts=FAKE, n=FAKE, u=FAKE, B=4, K=2, V=100, tokens=FAKE, counts=FAKE, ws=FAKE, bytes=1 << 40)
    v.update(kw)
    return lib.isst_op_verify_drafts(v["t"], v["ts"], v["tr"], v["q"], v["qs"], v["qr"], v["drafts"], v["n"], v["u"], v["B"], v["K"], v["V"], v["tokens"], v["counts"], v["ws"],
                                     v["bytes"], None)


@pytest.mark.parametrize("bad", [dict(t=None), dict(drafts=None), dict(tokens=None), dict(counts=None), dict(ws=None), dict(ws=FAKE + 8), dict(B=-1), dict(K=-1), dict(V=0), dict(ts=-1),
                                 dict(qr=-1), dict(B=1 << 24), dict(t=FAKE + 2), dict(u=FAKE + 4)])
def test_verify_drafts_refuses(lib, bad):
    assert verify(lib, **bad) == -1


def test_verify_drafts_workspace(lib):
    need = lib.isst_op_verify_drafts_workspace(4, 2, 100)
    assert need > 0 and verify(lib, bytes=need - 1) == -4 and verify(lib, B=0) == 0
    assert lib.isst_op_verify_drafts_workspace(4, 2, 0) == -1


def test_python_functions_refuse_cpu_tensors_and_wrong_kinds(lib):
    bf, i32 = torch.bfloat16, torch.int32
    q, k, t, ln = torch.zeros(2, 4, 128, dtype=bf), torch.zeros(2, 9, 128, dtype=bf), torch.zeros(2, 2, 8, 128, dtype=bf), torch.zeros(2, dtype=i32)
    with pytest.raises(E.IsstError, match="GPU"):
        E.op_prefix_attention(q, k, k, t, t, ln)
    with pytest.raises(E.IsstError, match="GPU"):
        E.op_gemm_lora(torch.zeros(2, 32, dtype=bf), torch.zeros(512, dtype=bf), 16, torch.zeros(1, 8, 32, dtype=bf), torch.zeros(1, 16, 8, dtype=bf), torch.zeros(1), ln)
    with pytest.raises(E.IsstError, match="GPU"):
        E.op_verify_drafts(torch.zeros(2, 3, 5), torch.zeros(2, 2, dtype=i32))
    # (checks behind the device's: on shapes and kinds alone)
    with pytest.raises(E.IsstError, match="must be torch.bfloat16"):
        E._expect("op", -1, "q", q.float(), bf, (2, 4, 128))
    with pytest.raises(E.IsstError, match="must be torch.bfloat16"):
        E._expect("op", -1, "q", q, bf, (2, 4, 64))
    with pytest.raises(E.IsstError, match="expected cuda:0"):
        E._expect("op", 0, "q", q, bf, (2, 4, 128))
    with pytest.raises(E.IsstError, match="contiguous"):
        E._expect("op", -1, "x", torch.zeros(4, 6).t(), torch.float32, (6, 4))
    for view in (q.transpose(1, 2), torch.zeros(2, 4, 132, dtype=bf)[:, :, :128], torch.zeros(2 * 4 * 128 + 1, dtype=bf)[1:].view(2, 4, 128)):
        with pytest.raises(E.IsstError, match="16-byte aligned"):
            E._row_strides("op", "q", view)
    odd = torch.zeros(1, 2, 129, dtype=bf)[:, :1, :128]  # strides of dims without a second entry do not count
    assert E._row_strides("op", "q", q) == (512, 128) and E._row_strides("op", "q", odd) == (0, 0) and E._row_strides("op", "k", odd[:, :0]) == (0, 0)
