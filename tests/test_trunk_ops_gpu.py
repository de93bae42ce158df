"""Attention, query / key norm with rotation and embedding as a program uses them: through torch.ops.lrce with autograd, in a
run, on other streams, captured, with masked rubbish, unusual strides, empty sizes and long caches."""
import math

import pytest
import torch

from attention_ref import check, reference

pytestmark = pytest.mark.gpu
dev = "cuda"
F64 = torch.float64
BF = torch.bfloat16


def K():
    from lrce import kernels
    return kernels


def ops():
    from lrce import ops  # noqa: F401  (registers the ops)
    return torch.ops.lrce


def rnd(seed, *shape, dtype=BF):
    return torch.randn(*shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def both(q, k, v, do, m, causal=False):
    out, lse = K().attention(q, k, v, key_mask=m, causal=causal)
    return (out, lse, *K().attention_bwd(do, q, k, v, out, lse, key_mask=m, causal=causal))


@pytest.mark.parametrize("Lq,Lk,D", [(70, 333, 64), (1, 700, 128), (300, 200, 32), (33, 1500, 96)])
def test_hidden_keys_may_hold_anything(Lq, Lk, D):
    q, k, v, do = rnd(1, 2, Lq, 4, D), rnd(2, 2, Lk, 2, D), rnd(3, 2, Lk, 2, D), rnd(4, 2, Lq, 4, D)
    m = torch.rand(2, Lk, generator=torch.Generator(device=dev).manual_seed(9), device=dev) < 0.5
    m[0, Lk // 2:] = False
    for causal in (False, True):
        clean = both(q, k, v, do, m, causal)
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(BF).min):
            kb, vb = (torch.where(m[:, :, None, None], t, torch.full_like(t, bad)) for t in (k, v))
            for a, b in zip(both(q, kb, vb, do, m, causal), clean):
                assert torch.equal(a, b), (bad, causal)


def test_nan_and_infinity_that_are_seen_are_not_lost():
    q, k, v = rnd(1, 1, 5, 2, 64), rnd(2, 1, 600, 2, 64), rnd(3, 1, 600, 2, 64)
    v[0, 77, 1] = math.nan
    k[0, 400, 0, 3] = math.nan
    for L in (1, 5):
        out, lse = K().attention(q[:, :L], k, v)
        assert torch.isnan(out[0, :, 1]).all() and torch.isnan(out[0, :, 0]).all() and torch.isnan(lse[0, 0]).all()
        assert torch.isfinite(lse[0, 1]).all()


def test_strides_and_alignment():
    B, L, H, Hk, D = 2, 90, 4, 2, 64
    q0, k0, v0, do0 = rnd(1, B, H, L, D), rnd(2, B, Hk, L, D), rnd(3, B, Hk, L, D), rnd(4, B, H, L, D)
    q, k, v, do = (t.transpose(1, 2) for t in (q0, k0, v0, do0))            # head-major storage
    want = both(*(t.contiguous() for t in (q, k, v, do)), None)
    for a, b in zip(both(q, k, v, do, None), want):
        assert torch.equal(a, b)
    odd = torch.empty(B * L * H * D + 1, dtype=BF, device=dev)[1:].view(B, L, H, D)   # not at a 16-byte boundary
    odd.copy_(q)
    for a, b in zip(both(odd, k, v, do, None), want):
        assert torch.equal(a, b)
    wide = torch.empty(B, L, H, D + 3, dtype=BF, device=dev)[..., 1:D + 1]              # odd row pitch
    wide.copy_(q)
    for a, b in zip(both(wide, k, v, do, None), want):
        assert torch.equal(a, b)
    one = k[:1].expand(B, L, Hk, D)                                                     # one memory for the batch (stride 0)
    for a, b in zip(both(q, one, one, do, None), both(q, one.contiguous(), one.contiguous(), do, None)):
        assert torch.equal(a, b)
    m = (torch.arange(2 * L, device=dev) % 5 > 0)[None].expand(B, 2 * L)[:, ::2]        # strided, expanded mask
    for a, b in zip(both(q, k, v, do, m), both(q, k, v, do, m.contiguous())):
        assert torch.equal(a, b)


def test_empty_sizes():
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 0, 0), (2, 1, 0)):
        q, k, do = rnd(1, B, Lq, 4, 32), rnd(2, B, Lk, 2, 32), rnd(3, B, Lq, 4, 32)
        m = torch.ones(B, Lk, dtype=torch.bool, device=dev)
        for mask in (None, m):
            out, lse, dq, dk, dv = both(q, k, k, do, mask)
            torch.cuda.synchronize()
            assert (out == 0).all() and (lse == -math.inf).all() and (dq == 0).all() and (dk == 0).all() and (dv == 0).all()
            assert dk.shape == k.shape and dq.shape == q.shape
    w, f = torch.ones(32, device=dev), torch.ones(16, device=dev)
    for B, L in ((0, 3), (2, 0)):
        q, k = rnd(1, B, L, 4, 32), rnd(2, B, L, 2, 32)
        pos = torch.zeros(B, L, dtype=torch.int64, device=dev)
        assert K().qk_norm_rope(q, k, w, w, pos, f)[0].shape == q.shape
        dq, dk, dqw, dkw = K().qk_norm_rope_bwd(q, k, q, k, w, w, pos, f)
        assert (dqw == 0).all() and (dkw == 0).all()


def test_masks_that_see_one_key_or_none_at_the_ends():
    """The only visible key is the first, the last, or at a tile's border; causal rows before the first key see none."""
    for at in (0, 63, 64, 199):
        m = torch.zeros(2, 200, dtype=torch.int32, device=dev)
        m[0, at] = 1
        for Lq in (1, 50, 260):
            q, k, v, do = rnd(1, 2, Lq, 2, 64), rnd(2, 2, 200, 2, 64), rnd(3, 2, 200, 2, 64), rnd(4, 2, Lq, 2, 64)
            for causal in (False, True):
                got = dict(zip(("out", "lse", "dq", "dk", "dv"), both(q, k, v, do, m, causal)))
                check(got, reference(q, k, v, m, causal, None, do), f"{at} {Lq} {causal}")


def test_large_scores():
    """Scores of some hundreds: the running maximum rises by more than its slack, later keys win and lose."""
    q, k, v, do = (rnd(i, 1, 150, 2, 64, dtype=torch.float16) for i in (1, 2, 3, 4))
    k = (k * torch.linspace(0.5, 30, 150, device=dev)[None, :, None, None]).half()
    for kk in (k, k.flip(1)):
        for causal in (False, True):
            got = dict(zip(("out", "lse", "dq", "dk", "dv"), both(q, kk, v, do, None, causal)))
            check(got, reference(q, kk, v, None, causal, None, do), "large scores")
        got = dict(zip(("out", "lse"), K().attention(q[:, -1:], kk, v)))
        check(got, reference(q[:, -1:], kk, v), "large scores, one row")


def test_backward_does_not_depend_on_timing():
    for B, Lq, Lk, H, Hk in ((1, 3000, 257, 8, 1), (2, 200, 200, 4, 4)):
        q, k, v, do = rnd(1, B, Lq, H, 64), rnd(2, B, Lk, Hk, 64), rnd(3, B, Lk, Hk, 64), rnd(4, B, Lq, H, 64)
        first = both(q, k, v, do, None)
        for _ in range(3):
            for a, b in zip(both(q, k, v, do, None), first):
                assert torch.equal(a, b)


def test_gradients_against_differences():
    """Central differences of the 64-bit forward along single coordinates."""
    q, k, v, do = rnd(1, 1, 20, 4, 32), rnd(2, 1, 30, 2, 32), rnd(3, 1, 30, 2, 32), rnd(4, 1, 20, 4, 32)
    m = torch.arange(30, device=dev)[None] != 7
    _, _, dq, dk, dv = both(q, k, v, do, m, True)
    allow = reference(q, k, v, m, True, None, do)

    def loss(a, b, c):
        ok = m[0] & (torch.arange(30, device=dev)[None] <= torch.arange(20, device=dev)[:, None] + 10)
        s = (a.transpose(1, 2) @ b.repeat_interleave(2, 2).permute(0, 2, 3, 1)) * 32 ** -0.5
        p = s.masked_fill(~ok, -math.inf).softmax(-1)
        return ((p @ c.repeat_interleave(2, 2).transpose(1, 2)).transpose(1, 2) * do.to(F64)).sum()

    x = [t.to(F64) for t in (q, k, v)]
    h = 1e-4
    g = torch.Generator().manual_seed(3)
    for i, (name, got) in enumerate((("dq", dq), ("dk", dk), ("dv", dv))):
        for _ in range(25):
            at = tuple(int(torch.randint(n, (1,), generator=g)) for n in got.shape)
            ends = []
            for sgn in (1, -1):
                y = [t.clone() for t in x]
                y[i][at] += sgn * h
                ends.append(loss(*y))
            fd = ((ends[0] - ends[1]) / (2 * h)).item()
            assert abs(got[at].item() - fd) <= allow[name][1][at].item() + 1e-6, (name, at)   # 1e-6: the difference's own h^2 and rounding


def test_a_cache_past_32_bit_offsets():
    L, Hk, D = 70000, 256, 128                                              # 2.3e9 elements: 4.6 GB each
    k = torch.empty(1, L, Hk, D, dtype=BF, device=dev)
    v = torch.empty(1, L, Hk, D, dtype=BF, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    for t in (k, v):
        for part in t[0].split(10000):
            part.copy_(torch.randn(part.shape, generator=g, device=dev, dtype=torch.float32))
    q = rnd(2, 1, 1, Hk, D)
    out, lse = K().attention(q, k, v)
    hs = slice(Hk - 2, Hk)
    check({"out": out[:, :, hs], "lse": lse[:, hs]}, reference(q[:, :, hs], k[:, :, hs], v[:, :, hs]), "last heads")
    q = rnd(3, 1, 40, 2, D)
    do = rnd(4, 1, 40, 2, D)
    got = dict(zip(("out", "lse", "dq", "dk", "dv"), both(q, k[:, :, hs], v[:, :, hs], do, None)))
    check(got, reference(q, k[:, :, hs], v[:, :, hs], None, False, None, do), "rows 64 KB apart")


def block(ids, table, w_qkv, qw, kw, freq, w_out, H, Hk, D, pad):
    """embedding -> linear -> norm + rotation -> causal attention -> linear, through torch.ops.lrce"""
    o = ops()
    B, L = ids.shape
    x = o.embedding(ids, table, 4.0, 0)
    qkv = o.linear(x.view(B * L, -1), w_qkv).view(B, L, H + 2 * Hk, D)
    q, k, v = qkv.split([H, Hk, Hk], 2)
    pos = torch.arange(L, device=dev)
    q, k = o.qk_norm_rope(q, k, qw, kw, pos, freq, 1e-6, False)
    y, _ = o.attention(q, k, v, pad, True)
    return o.linear(y.reshape(B * L, H * D), w_out)


def block_ref(ids, table, w_qkv, qw, kw, freq, w_out, H, Hk, D, pad):
    B, L = ids.shape
    x = torch.nn.functional.embedding(ids, table, padding_idx=0) * 4.0
    q, k, v = (x.view(B * L, -1) @ w_qkv.t()).view(B, L, H + 2 * Hk, D).split([H, Hk, Hk], 2)
    ang = torch.arange(L, device=dev, dtype=F64)[:, None, None] * freq.to(F64)

    def rope(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = t.chunk(2, -1)
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)

    q, k, v = (t.transpose(1, 2) for t in (rope(q, qw), rope(k, kw).repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)))
    ok = pad[:, None, None, :] & torch.ones(L, L, dtype=torch.bool, device=dev).tril()
    p = (q @ k.transpose(-1, -2) * D ** -0.5).masked_fill(~ok, -math.inf).softmax(-1)
    return (p @ v).transpose(1, 2).reshape(B * L, H * D) @ w_out.t()


def chain(seed=0, B=3, L=75, C=192, H=6, Hk=2, D=64, V=500):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)
    ids = torch.randint(1, V, (B, L), generator=g, device=dev)
    pad = torch.ones(B, L, dtype=torch.bool, device=dev)
    ids[1, 50:], pad[1, 50:] = 0, False
    leaves = [(r(V, C) * 0.5).to(BF), (r((H + 2 * Hk) * D, C) / C ** 0.5).to(BF), 1 + 0.2 * r(D), 1 + 0.2 * r(D), (r(C, H * D) / (H * D) ** 0.5).to(BF)]
    freq = 100.0 ** (-torch.arange(D // 2, device=dev) * 2.0 / D)
    return ids, leaves, freq, (H, Hk, D, pad), r(B * L, C)


def test_a_run_of_them_with_autograd():
    ids, leaves, freq, cfg, R = chain()
    t, wq, qw, kw, wo = [x.clone().requires_grad_() for x in leaves]
    y = block(ids, t, wq, qw, kw, freq, wo, *cfg)
    (y.float() * R).sum().backward()
    ref = [x.to(F64).requires_grad_() for x in leaves]
    yr = block_ref(ids, ref[0], ref[1], ref[2], ref[3], freq, ref[4], *cfg)
    (yr * R.to(F64)).sum().backward()
    rel = lambda a, b: ((a.to(F64) - b).norm() / b.norm()).item()
    # at most twelve values on the way are rounded to bf16 (half a step, 2^-8 of the value, each)
    assert rel(y, yr) <= 12 * 2.0 ** -8
    for got, want in zip((t, wq, qw, kw, wo), ref):
        assert got.grad.dtype == got.dtype and rel(got.grad, want.grad) <= 12 * 2.0 ** -8, tuple(got.shape)
    assert (t.grad[0] == 0).all()                                            # padding


def test_only_some_gradients():
    """Outputs and inputs that take no part in the backward."""
    q, k = rnd(1, 1, 6, 2, 32).requires_grad_(), rnd(2, 1, 6, 2, 32).requires_grad_()
    w, f, pos = torch.ones(32, device=dev), torch.ones(16, device=dev), torch.arange(6, device=dev)
    a, _ = ops().qk_norm_rope(q, k, w, w, pos, f, 1e-6, False)
    a.float().sum().backward()
    assert torch.isfinite(q.grad).all() and (k.grad is None or (k.grad == 0).all())
    q2 = rnd(3, 1, 6, 2, 32).requires_grad_()
    out, lse = ops().attention(q2, k.detach(), k.detach())
    assert not lse.requires_grad
    out.float().sum().backward()
    assert torch.isfinite(q2.grad).all()


def everything(ids, leaves, freq, cfg, R):
    """Forward and backward by the kernels' own calls: what a captured step does."""
    H, Hk, D, pad = cfg
    table, wq, qw, kw, wo = leaves
    B, L = ids.shape
    k_ = K()
    x = k_.embedding(ids, table, scale=4.0)
    q, k, v = k_.linear(x.view(B * L, -1), wq).view(B, L, H + 2 * Hk, D).split([H, Hk, Hk], 2)
    pos = torch.arange(L, device=dev)
    qr, kr = k_.qk_norm_rope(q, k, qw, kw, pos, freq)
    out, lse = k_.attention(qr, kr, v, key_mask=pad, causal=True)
    do = R.to(BF).view(B, L, -1)[..., :1].unsqueeze(2) * out
    dq, dk, dv = k_.attention_bwd(do, qr, kr, v, out, lse, key_mask=pad, causal=True)
    gq, gk, gqw, gkw = k_.qk_norm_rope_bwd(dq, dk, q, k, qw, kw, pos, freq)
    dw = k_.embedding_bwd(x, ids, table.shape[0], scale=4.0, padding_idx=0)
    long, _ = k_.attention(qr[:, -1:], kr.repeat(1, 40, 1, 1), v.repeat(1, 40, 1, 1))   # few rows over many keys: split and joined
    return out, lse, dv, gq, gk, gqw, gkw, dw, long


def test_captured_and_replayed():
    ids, leaves, freq, cfg, R = chain()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        everything(ids, leaves, freq, cfg, R)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = everything(ids, leaves, freq, cfg, R)
    with torch.cuda.graph(other):                                            # a second one beside it: own workspaces
        got2 = everything(ids, leaves, freq, cfg, R)
    for seed in (1, 2, 3):
        ids2, leaves2, _, _, R2 = chain(seed)
        keep = ids == 0
        ids.copy_(ids2.masked_fill(keep, 0))
        for a, b in zip(leaves, leaves2):
            a.copy_(b)
        R.copy_(R2)
        want = [t.clone() for t in everything(ids, leaves, freq, cfg, R)]
        for g_, outs in ((graph, got), (other, got2), (graph, got)):
            for t in outs:
                t.fill_(7)
            g_.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_captured_autograd_step():
    """Forward and backward of the operators in one graph, whose leaves no eager graph holds."""
    ids, leaves, freq, cfg, R = chain(5)
    live = [x.clone().requires_grad_() for x in leaves]

    def step():
        y = block(ids, live[0], live[1], live[2], live[3], freq, live[4], *cfg)
        return torch.autograd.grad((y.float() * R).sum(), live)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_on_other_streams_at_once():
    ids, leaves, freq, cfg, R = chain(7)
    want = [t.clone() for t in everything(ids, leaves, freq, cfg, R)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(everything(ids, leaves, freq, cfg, R))
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


def test_refusals():
    from lrce import _native as N
    k_ = K()
    q, k = rnd(1, 2, 5, 4, 64), rnd(2, 2, 7, 2, 64)
    out, lse = k_.attention(q, k, k)
    w, f, pos = torch.ones(64, device=dev), torch.ones(32, device=dev), torch.arange(5, device=dev)
    k5 = k[:, :5]
    ids, table = torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(4, 8, device=dev)
    bad = [
        lambda: k_.attention(q.float(), k.float(), k.float()), lambda: k_.attention(q, k, k[:, :6]), lambda: k_.attention(q, k.half(), k),
        lambda: k_.attention(q[0], k, k), lambda: k_.attention(rnd(1, 2, 5, 4, 48), rnd(1, 2, 5, 4, 48), rnd(1, 2, 5, 4, 48)),
        lambda: k_.attention(q[:, :, :3], k, k), lambda: k_.attention(q[:1], k, k), lambda: k_.attention(q, k, k, scale=-1.0),
        lambda: k_.attention(q, k, k, key_mask=torch.ones(2, 6, dtype=torch.bool, device=dev)),
        lambda: k_.attention(q, k, k, key_mask=torch.ones(2, 7, device=dev)), lambda: k_.attention(q, k, k, key_mask=torch.ones(2, 7, dtype=torch.bool)),
        lambda: k_.attention_bwd(q[:, :4], q, k, k, out, lse), lambda: k_.attention_bwd(q, q, k, k, out, lse[:, :, :4]),
        lambda: k_.attention_bwd(q, q, k, k, out, lse.double()),
        lambda: k_.qk_norm_rope(q, k, w, w, pos, f), lambda: k_.qk_norm_rope(q, k5, w[:32], w, pos, f), lambda: k_.qk_norm_rope(q, k5, w.half(), w, pos, f),
        lambda: k_.qk_norm_rope(q, k5, w, w, pos.float(), f), lambda: k_.qk_norm_rope(q, k5, w, w, pos[:4], f),
        lambda: k_.qk_norm_rope(q, k5, w, w, pos, torch.ones(33, device=dev)), lambda: k_.qk_norm_rope(q, k5, w, w, pos, f, eps=-1.0),
        lambda: k_.qk_norm_rope_bwd(q, q, q, k5, w, w, pos, f),
        lambda: k_.embedding(ids.float(), table), lambda: k_.embedding(ids, table.bfloat16(), out_dtype=torch.float32),
        lambda: k_.embedding(ids, table[0]), lambda: k_.embedding(ids.cpu(), table),
        lambda: k_.embedding_bwd(table, ids, 4), lambda: k_.embedding_bwd(table[:3], ids, 0), lambda: k_.embedding_bwd(table[:3], ids, 4, dw=table[:3]),
        lambda: k_.embedding_bwd(table[:3], ids, 4, dw=torch.zeros(8, 4, device=dev).t()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(N.NativeError):
            call()
            pytest.fail(f"call {i} was accepted")


@pytest.mark.parametrize("Lq,Lk,H,D", [(1, 20000, 8, 64), (1, 600, 8, 64), (3, 700, 4, 128), (300, 600, 4, 32), (900, 64, 4, 64)])
def test_what_is_seen_under_a_weight_of_zero_is_not_lost(Lq, Lk, H, D):
    """A visible v of NaN or infinity whose key lies 128 below the row's maximum (a weight of 0 in 32 bits): 0 x NaN, by whatever split
    of the keys - shares joined, waves joined, one walk."""
    q = torch.full((1, Lq, H, D), 4.0, dtype=BF, device=dev)
    k, v = torch.zeros(1, Lk, 2, D, dtype=BF, device=dev), rnd(1, 1, Lk, 2, D)
    k[:, -1] = 128 / (4.0 * D ** 0.5)
    for bad in (math.nan, math.inf):
        w = v.clone()
        w[0, 3, 1, 5] = bad
        out, lse = K().attention(q, k, w)
        assert not torch.isfinite(out[0, :, H // 2:, 5]).any()
        out[0, :, H // 2:, 5] = 0
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        m = torch.ones(1, Lk, dtype=torch.bool, device=dev)
        m[0, 3] = False
        assert torch.isfinite(K().attention(q, k, w, key_mask=m)[0]).all()


def operator_calls():
    g = torch.Generator(device=dev).manual_seed(21)
    q, k, v = rnd(1, 2, 40, 4, 64), rnd(2, 2, 70, 2, 64), rnd(3, 2, 70, 2, 64)
    m = torch.rand(2, 70, generator=g, device=dev) < 0.7
    w, kw, f = rnd(4, 64, dtype=torch.float32), rnd(5, 64, dtype=torch.float32), torch.linspace(1, 0.01, 20, device=dev)
    pos, ids = torch.arange(40, device=dev), torch.randint(0, 50, (2, 40), generator=g, device=dev)
    return (("attention", (q, k, v, m, True, 0.2)), ("qk_norm_rope", (q, k[:, :40], w, kw, pos, f, 1e-5, True)),
            ("embedding", (ids, rnd(6, 50, 64), 2.0, 3)))


def test_autograd_is_the_backward_calls():
    """The gradients that autograd hands out are the backward calls' own, bit for bit; integers, masks and frequencies have none."""
    for name, args in operator_calls():
        live = [a.clone().requires_grad_() if torch.is_tensor(a) and a.is_floating_point() else a for a in args]
        if name == "qk_norm_rope":
            live[5] = args[5]
        y = getattr(ops(), name)(*live)
        outs = [t for t in (y if isinstance(y, tuple) else (y,)) if t.requires_grad]
        dy = [rnd(30 + i, *t.shape, dtype=t.dtype) for i, t in enumerate(outs)]
        got = torch.autograd.grad(outs, [t for t in live if torch.is_tensor(t) and t.requires_grad], dy)
        if name == "attention":
            q, k, v, m, causal, scale = args
            want = K().attention_bwd(dy[0], q, k, v, *K().attention(q, k, v, m, causal, scale), m, causal, scale)
        elif name == "qk_norm_rope":
            want = K().qk_norm_rope_bwd(*dy, *args)
        else:
            want = (K().embedding_bwd(dy[0], args[0], 50, args[2], args[3]).to(BF),)
        assert len(got) == len(want)
        for a, b in zip(got, want):
            assert a.dtype == b.dtype and torch.equal(a, b), name


def test_operators_keep_the_dispatchers_rules():
    """Schemas, shapes without data, and autograd by torch's own check."""
    for name, args in operator_calls():
        live = [a.clone().requires_grad_() if torch.is_tensor(a) and a.is_floating_point() and a.dim() > 1 else a for a in args]
        torch.library.opcheck(getattr(ops(), name).default, tuple(live))
