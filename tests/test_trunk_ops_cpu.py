"""Attention, query / key norm with rotation and embedding without a GPU: the C entry points' refusals (no launch), the
wrappers' refusals of CPU tensors, the operators' schemas and shapes."""
import ctypes

import pytest
import torch

A = 0x7F0000000000                                            # an address nobody reads


def lib():
    from lrce import _native as N
    return N, N.lib()


def attn(**over):
    N, _ = lib()
    d = N.AttnDesc()
    d.q = d.k = d.v = d.out = d.lse = A
    d.B, d.H, d.Hk, d.Lq, d.Lk, d.D, d.scale = 2, 4, 2, 8, 8, 64, 0.125
    for n, h in (("q", 4), ("k", 2), ("v", 2), ("o", 4)):
        setattr(d, f"{n}_sb", 8 * h * 64), setattr(d, f"{n}_sl", h * 64), setattr(d, f"{n}_sh", 64)
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,word", [
    (dict(Hk=3), b"query heads"), (dict(D=48), b"head dim"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(Lq=-1), b"sizes"), (dict(H=0), b"sizes"), (dict(q=None), b"null"), (dict(k=None), b"null"),
    (dict(k_sl=100), b"multiples of 8"), (dict(v=A + 8), b"16 bytes"), (dict(k_sl=1 << 23), b"stride"), (dict(key_mask=A, mask_bytes=2), b"mask"),
    (dict(Lk=1 << 30), b"long"), (dict(B=1 << 28, Lq=1 << 12), b"rows")])
def test_attention_refusals(over, word):
    _, L = lib()
    for fn in (L.lrce_attn_fwd, L.lrce_attn_bwd):
        assert fn(ctypes.byref(attn(**over)), None) == 1
        assert word in L.lrce_last_error(), L.lrce_last_error()
    assert L.lrce_attn_fwd_workspace(ctypes.byref(attn(**over))) == -1
    assert L.lrce_attn_bwd_workspace(ctypes.byref(attn(**over))) == -1


def test_attention_null_descriptor_and_workspace():
    _, L = lib()
    assert L.lrce_attn_fwd(None, None) == 1 and L.lrce_attn_bwd(None, None) == 1
    d = attn(Lq=1, Lk=100000, B=1, H=2)                       # few rows, many keys: the partials need room
    assert L.lrce_attn_fwd_workspace(ctypes.byref(d)) > 0
    assert L.lrce_attn_fwd(ctypes.byref(d), None) == 1 and b"workspace" in L.lrce_last_error()
    d = attn(Lq=100)                                           # (up to 64 queries and keys need none)
    d.dout = d.dq = d.dk = d.dv = A
    assert L.lrce_attn_bwd(ctypes.byref(d), None) == 1 and b"workspace" in L.lrce_last_error()
    d.dk = None
    assert L.lrce_attn_bwd(ctypes.byref(d), None) == 1 and b"null gradient" in L.lrce_last_error()
    d = attn(B=0)
    assert L.lrce_attn_fwd(ctypes.byref(d), None) == 0        # nothing to do
    assert L.lrce_attn_fwd_workspace(ctypes.byref(d)) == 0


def rope(**over):
    N, _ = lib()
    d = N.RopeDesc()
    d.q = d.k = d.q_weight = d.k_weight = d.positions = d.inv_freq = d.q_out = d.k_out = A
    d.B, d.L, d.H, d.Hk, d.D, d.R, d.pos_bytes, d.eps = 1, 4, 2, 1, 64, 64, 8, 1e-6
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,word", [
    (dict(D=12), b"head dim"), (dict(D=264), b"head dim"), (dict(R=65), b"rotated"), (dict(R=3), b"rotated"), (dict(R=0), b"rotated"),
    (dict(dtype=3), b"dtype"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(pos_bytes=2), b"positions"),
    (dict(H=0), b"sizes"), (dict(q=None), b"null"), (dict(inv_freq=None), b"null"), (dict(positions=None), b"null")])
def test_rope_refusals(over, word):
    _, L = lib()
    assert L.lrce_qk_norm_rope_fwd(ctypes.byref(rope(**over)), None) == 1
    assert word in L.lrce_last_error(), L.lrce_last_error()
    d = rope(gq=A, gk=A, dq_weight=A, dk_weight=A, **over)
    assert L.lrce_qk_norm_rope_bwd(ctypes.byref(d), None) == 1 and word in L.lrce_last_error()


def test_rope_workspace():
    _, L = lib()
    for tokens, D in ((-1, 64), (4, 12), (4, 264), (4, 0)):
        assert L.lrce_qk_norm_rope_bwd_workspace(tokens, D) == -1
    assert L.lrce_qk_norm_rope_bwd_workspace(0, 64) == 128


def test_rope_backward_needs_gradients_and_a_workspace():
    _, L = lib()
    assert L.lrce_qk_norm_rope_bwd(ctypes.byref(rope()), None) == 1 and b"gradient" in L.lrce_last_error()
    d = rope(gq=A, gk=A, dq_weight=A, dk_weight=A)
    assert L.lrce_qk_norm_rope_bwd(ctypes.byref(d), None) == 1 and b"workspace" in L.lrce_last_error()
    assert L.lrce_qk_norm_rope_fwd(ctypes.byref(rope(B=0)), None) == 0


def test_embedding_refusals():
    _, L = lib()
    ok = dict(ids=A, ib=8, n=4, w=A, ld=16, rows=10, cols=16, wt=2, y=A, yt=2)

    def fwd(**o):
        a = {**ok, **o}
        return L.lrce_embedding_fwd(a["ids"], a["ib"], a["n"], a["w"], a["ld"], a["rows"], a["cols"], a["wt"], a["y"], a["yt"], 1.0, None)

    for o, word in ((dict(ib=2), b"ids"), (dict(n=-1), b"sizes"), (dict(rows=0), b"sizes"), (dict(rows=1 << 31), b"sizes"), (dict(cols=0), b"sizes"),
                    (dict(wt=0, yt=2), b"types"), (dict(wt=3), b"types"), (dict(ld=8), b"pitch"), (dict(ids=None), b"null"), (dict(y=None), b"null")):
        assert fwd(**o) == 1 and word in L.lrce_last_error(), (o, L.lrce_last_error())
    assert fwd(n=0, ids=None) == 0
    ok = dict(ids=A, ib=8, n=4, dy=A, dt=2, dw=A, rows=10, cols=16, ws=None, k=0)

    def bwd(**o):
        a = {**ok, **o}
        return L.lrce_embedding_bwd(a["ids"], a["ib"], a["n"], a["dy"], a["dt"], a["dw"], a["rows"], a["cols"], 1.0, -1, 1, a["ws"], a["k"], None)

    for o, word in ((dict(ib=1), b"ids"), (dict(n=1 << 31), b"sizes"), (dict(dt=5), b"type"), (dict(dw=A + 4), b"16 bytes"), (dict(dw=None), b"16 bytes"),
                    (dict(dy=None), b"null"), (dict(n=4000), b"workspace"), (dict(n=4000, ws=A + 4, k=1 << 20), b"workspace")):
        assert bwd(**o) == 1 and word in L.lrce_last_error(), (o, L.lrce_last_error())
    assert bwd(n=0) == 0
    assert L.lrce_embedding_bwd_workspace(-1, 10, 16) == -1 and L.lrce_embedding_bwd_workspace(4000, 10, 16) > 0


def test_wrappers_refuse_cpu_tensors():
    from lrce import kernels as K, _native as N
    q = torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16)
    w, pos, f, ids = torch.ones(64), torch.zeros(2, dtype=torch.int64), torch.ones(32), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: K.attention(q, q, q), lambda: K.attention_bwd(q, q, q, q, q, torch.zeros(1, 2, 2)),
                 lambda: K.qk_norm_rope(q, q, w, w, pos, f), lambda: K.qk_norm_rope_bwd(q, q, q, q, w, w, pos, f),
                 lambda: K.embedding(ids, torch.zeros(4, 8)), lambda: K.embedding_bwd(torch.zeros(3, 8), ids, 4)):
        with pytest.raises(N.NativeError, match="HIP device"):
            call()


def test_operators_shapes():
    from lrce import ops  # noqa: F401  (registers the ops)
    m = dict(device="meta")
    q, k = torch.empty(2, 5, 8, 64, dtype=torch.bfloat16, **m), torch.empty(2, 7, 2, 64, dtype=torch.bfloat16, **m)
    out, lse = torch.ops.lrce.attention(q, k, k, None, True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (2, 8, 5) and lse.dtype == torch.float32
    dq, dk, dv = torch.ops.lrce.attention_backward(out, q, k, k, out, lse, None, True)
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
    w, f = torch.empty(64, **m), torch.empty(32, **m)
    pos = torch.empty(2, 5, dtype=torch.int64, **m)
    k5 = k[:, :5]
    a, b = torch.ops.lrce.qk_norm_rope(q, k5, w, w, pos, f)
    assert a.shape == q.shape and b.shape == k5.shape
    assert [t.shape for t in torch.ops.lrce.qk_norm_rope_backward(a, b, q, k5, w, w, pos, f)] == [q.shape, k5.shape, w.shape, w.shape]
    ids = torch.empty(3, 4, dtype=torch.int32, **m)
    y = torch.ops.lrce.embedding(ids, torch.empty(100, 24, dtype=torch.float16, **m), 2.0)
    assert y.shape == (3, 4, 24) and y.dtype == torch.float16
    dw = torch.ops.lrce.embedding_backward(y, ids, 100)
    assert dw.shape == (100, 24) and dw.dtype == torch.float32


def test_padding_idx_is_a_row_or_none():
    """-1: none; what nn.Embedding would count from the end, or refuse, is refused."""
    from lrce import _native as N
    from lrce import ops  # noqa: F401  (registers the ops)
    _, L = lib()
    for pad, rc in ((-2, 1), (-10, 1), (10, 1), (1 << 40, 1), (-1, 0), (0, 0), (9, 0)):
        assert L.lrce_embedding_bwd(A, 8, 0, A, 2, A, 10, 16, 1.0, pad, 1, None, 0, None) == rc, pad   # (no token: nothing is launched)
        assert rc == 0 or b"padding_idx" in L.lrce_last_error()
        if rc:
            with pytest.raises(N.NativeError, match="padding_idx"):
                torch.ops.lrce.embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(10, 16), 1.0, pad)
            with pytest.raises(N.NativeError, match="padding_idx"):
                torch.ops.lrce.embedding_backward(torch.zeros(3, 16), torch.zeros(3, dtype=torch.int64), 10, 1.0, pad)
