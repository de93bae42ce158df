"""Query / key norm with the position rotation (csrc/qk_rope.hip) and the embedding with its gradient by sorted tokens
(csrc/embedding.hip) through lrce.kernels, against 64-bit references, element by element within derived allowances."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
dev = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F64 = torch.float64
E32 = 2.0 ** -24


def K():
    from lrce import kernels
    return kernels


def near(got, want, allow, what):
    got = got.to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel():
        off = (got - want).abs()
        assert (off <= allow).all(), f"{what}: worst {(off / allow).nan_to_num(nan=math.inf).max().item():.3g} of the allowance"


# --------------------------------------------------------------------------------------------- norm + rotation
def rope_ref(x, w, pos, freq, eps, inter, dy=None):
    """{name: (value, allowance)} for one of q / k."""
    u = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else E32
    tiny = float(torch.finfo(x.dtype).tiny) * torch.finfo(x.dtype).eps
    B, L, H, D = x.shape
    R = 2 * freq.numel()
    X, W = x.to(F64), w.to(F64)
    pos = pos.expand(B, L)
    ang = pos.to(F64)[:, :, None, None] * freq.to(F64)
    cos, sin = ang.cos(), ang.sin()
    at = torch.arange(R, device=x.device)
    ia, ib = (at[0::2], at[1::2]) if inter else (at[:R // 2], at[R // 2:])

    def rot(z, sgn):
        y = z.clone()
        a, b = z[..., ia], z[..., ib]
        y[..., ia], y[..., ib] = a * cos - sgn * b * sin, b * cos + sgn * a * sin
        return y

    def both(z):                                              # |a| + |b| of the pair at both its places; elsewhere |z|
        y = z.abs().clone()
        y[..., ia] = y[..., ib] = z[..., ia].abs() + z[..., ib].abs()
        return y

    r = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = X * r
    y = rot(xh * W, 1)
    # the mean's D additions, the root, the products; the angle (6 units: its rounding in half turns, the sine's and cosine's)
    ops = (D + 24) * E32
    out = {"y": (y, ops * both(xh * W) + u * y.abs() + tiny)}
    if dy is None:
        return out
    g = rot(dy.to(F64), -1)
    ga = both(dy.to(F64))
    n = xh.abs() * ga
    gw = g * W
    m = (gw * xh).mean(-1, keepdim=True)
    dx = r * (gw - xh * m)
    scale = r * (ga * W.abs() + xh.abs() * (n * W.abs()).mean(-1, keepdim=True))
    out["dx"] = (dx, 2 * ops * scale + u * dx.abs() + tiny)
    # 128: a lane's rows, its exchanges, the waves, the workgroups' sums at these sizes
    out["dw"] = ((g * xh).sum((0, 1, 2)), (128 * E32 + 2 * ops) * n.sum((0, 1, 2)) + tiny)
    return out


def rope_case(B, L, H, Hk, D, R, dtype, inter, start=0, packed=True, flat_pos=False, pos_type=torch.int64, eps=1e-6, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev)
    if packed:
        q, k, _ = rn(B, L, H + 2 * Hk, D).to(DT[dtype]).split([H, Hk, Hk], 2)
    else:
        q, k = rn(B, L, H, D).to(DT[dtype]), rn(B, L, Hk, D).to(DT[dtype])
    qw, kw = 1 + 0.3 * rn(D), 1 + 0.3 * rn(D)
    pos = (start + torch.arange(L, device=dev)).to(pos_type)
    if not flat_pos:
        pos = torch.stack([pos + 3 * b for b in range(B)]) if B else pos.view(1, -1)[:0].expand(0, L)
    freq = (10000.0 ** (-torch.arange(R // 2, device=dev, dtype=F64) * 2 / R)).float()
    dq, dk = rn(B, L, H, D).to(DT[dtype]), rn(B, L, Hk, D).to(DT[dtype])
    yq, yk = K().qk_norm_rope(q, k, qw, kw, pos, freq, eps=eps, interleaved=inter)
    gq, gk, gqw, gkw = K().qk_norm_rope_bwd(dq, dk, q, k, qw, kw, pos, freq, eps=eps, interleaved=inter)
    torch.cuda.synchronize()
    what = f"{B}x{L}x{H}/{Hk}x{D} R={R} {dtype} inter={inter}"
    for n, x, w, y, d, dx, dw in (("q", q, qw, yq, dq, gq, gqw), ("k", k, kw, yk, dk, gk, gkw)):
        ref = rope_ref(x, w, pos, freq, eps, inter, d)
        near(y, *ref["y"], f"{what} {n}")
        near(dx, *ref["dx"], f"{what} d{n}")
        near(dw, *ref["dw"], f"{what} d{n}w")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,R", [(32, 32), (64, 64), (96, 32), (128, 128), (80, 80), (80, 40), (256, 256), (64, 6), (8, 2), (256, 10), (136, 70), (40, 40)])
def test_norm_rope(D, R, inter, dtype):
    rope_case(2, 37, 6, 2, D, R, dtype, inter)
    rope_case(3, 1, 4, 4, D, R, dtype, inter, start=131070, packed=False, flat_pos=True, pos_type=torch.int32)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (2, 5), (32, 8), (40, 1)])
def test_norm_rope_heads(H, Hk):
    rope_case(2, 150, H, Hk, 64, 64, "bf16", False, seed=1)
    rope_case(1, 9, H, Hk, 128, 64, "f32", True, seed=2, start=10 ** 6)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("eps", [0.0, 1e-50])
def test_norm_rope_without_eps(eps, dtype):
    """eps = 0, or one that is 0 in 32 bits: lanes without a head (12 of 16, 2 of 8) or without a token add nothing to the weights'
    gradients."""
    rope_case(2, 37, 12, 12, 64, 64, dtype, False, eps=eps)
    rope_case(2, 37, 8, 2, 128, 64, dtype, True, eps=eps)
    rope_case(1, 5, 1, 1, 32, 32, dtype, False, eps=eps)
    rope_case(1, 3, 3, 1, 136, 70, dtype, False, eps=eps)


@pytest.mark.parametrize("B,L,H,Hk,D,R,dtype,inter", [
    (2, 5003, 12, 2, 64, 64, "bf16", False), (2, 5003, 3, 3, 40, 40, "f16", True), (1, 9001, 4, 1, 96, 32, "f32", True), (1, 50011, 1, 1, 64, 64, "bf16", False)])
def test_norm_rope_of_more_tokens_than_are_resident(B, L, H, Hk, D, R, dtype, inter):
    """Over 4 x 768 (eight values a load) or 4 x 1024 waves' tokens: the backward's waves take several tokens each, the last ones fewer
    than the grid.  A weight gradient is then at most 4 tokens of one head in a lane, 6 exchanges, 3 waves and 16 + 6 sums of
    workgroups: below the 128 additions that the allowance counts."""
    rope_case(B, L, H, Hk, D, R, dtype, inter)


@pytest.mark.parametrize("inter", [False, True])
def test_rotation_of_far_positions(inter):
    """Rows whose only value is sqrt(64) (root mean square 1, each rounding but the angle's exact): the rotated pair is the cosine and the
    sine, each right to 3 units of its own size, near their zeros too.  The angle's three roundings in 64 bits, and the reference's
    one, are 4 x 2^-53 of it; 2^-44: the two terms of an angle's sine where they cancel."""
    L, D = 4001, 64
    pos = torch.cat([torch.arange(2000, device=dev), 2 ** 20 + 7 * torch.arange(2001, device=dev)])
    freq = (10000.0 ** (-torch.arange(32, device=dev, dtype=F64) / 32)).float()
    x = torch.zeros(1, L, 32, D, device=dev)
    first = 2 * torch.arange(32, device=dev) if inter else torch.arange(32, device=dev)
    second = first + (1 if inter else 32)
    x[0, :, torch.arange(32, device=dev), first] = 8.0
    w = torch.ones(D, device=dev)
    y, _ = K().qk_norm_rope(x, x[:, :, :1], w, w, pos, freq, eps=0.0, interleaved=inter)
    ang = pos.to(F64)[:, None] * freq.to(F64)
    i = torch.arange(32, device=dev)
    for got, want in ((y[0, :, i, first], ang.cos()), (y[0, :, i, second], ang.sin())):
        near(got / 8, want, 3 * 2.0 ** -23 * want.abs() + 4 * 2.0 ** -53 * ang + 2.0 ** -44, "cosine or sine")


def test_norm_rope_zero_rows_and_alignment():
    """Rows of zeros: the norm is held by eps; an odd start of the rows takes narrower loads, not wrong ones."""
    g = torch.Generator(device=dev).manual_seed(5)
    base = torch.randn(2, 5, 4 * 64 + 1, generator=g, device=dev).to(torch.bfloat16)
    q = base[..., 1:].unflatten(-1, (4, 64))                  # rows start at odd elements
    q[0, 0] = 0
    k = q[:, :, :1].clone()
    w = torch.ones(64, device=dev)
    pos = torch.arange(5, device=dev)
    freq = torch.linspace(1, 0.1, 32, device=dev)
    y, yk = K().qk_norm_rope(q, k, w, w, pos, freq)
    near(y, *rope_ref(q, w, pos, freq, 1e-6, False)["y"], "odd rows")
    near(yk, *rope_ref(k, w, pos, freq, 1e-6, False)["y"], "keys")
    assert (y[0, 0] == 0).all()


# --------------------------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("N,V,C", [(1, 5, 8), (17, 30, 1000), (320, 30522, 768), (512, 1, 4400), (512, 700, 9), (513, 700, 9), (1025, 7, 96), (8192, 4000, 33), (8193, 511, 64), (20011, 128000, 40),
                                   (40000, 3, 24)])
@pytest.mark.parametrize("types", [("f32", "f32", "f32"), ("bf16", "bf16", "bf16"), ("f16", "f16", "f32"), ("f32", "bf16", "f16")],
                         ids=lambda t: "-".join(t))
def test_embedding(N, V, C, types):
    g = torch.Generator(device=dev).manual_seed(N)
    w = torch.randn(V, C, generator=g, device=dev).to(DT[types[0]])
    ids = (V ** torch.rand(N, generator=g, device=dev, dtype=F64)).long().clamp_(0, V - 1)
    often = min(1, V - 1)
    ids[torch.rand(N, generator=g, device=dev) < 0.3] = often
    dy = torch.randn(N, C, generator=g, device=dev).to(DT[types[2]])
    for it, pad, scale in ((torch.int64, -1, 1.0), (torch.int32, often, 27.7)):
        i = ids.to(it)
        y = K().embedding(i, w, scale=scale, out_dtype=DT[types[1]])
        assert torch.equal(y, (w[ids].float() * scale).to(DT[types[1]]))
        got = K().embedding_bwd(dy, i, V, scale=scale, padding_idx=pad)
        again = K().embedding_bwd(dy, i, V, scale=scale, padding_idx=pad)
        assert torch.equal(got, again)
        keep = ids != pad
        ref, mag = torch.zeros(V, C, dtype=F64, device=dev), torch.zeros(V, C, dtype=F64, device=dev)
        d = dy.to(F64) * scale
        ref.index_put_((ids[keep],), d[keep], accumulate=True)
        mag.index_put_((ids[keep],), d[keep].abs(), accumulate=True)
        n = torch.bincount(ids, minlength=V).clamp(min=1).to(F64)[:, None]
        near(got, ref, (n.clamp(max=32 + N / 16) + 4) * E32 * mag, "dw")
        assert (got[~torch.isin(torch.arange(V, device=dev), ids[keep])] == 0).all()
        acc = torch.randn(V, C, generator=g, device=dev)
        was = acc.clone()
        back = K().embedding_bwd(dy, i, V, scale=scale, padding_idx=pad, dw=acc)
        assert back is acc and torch.equal(acc, was + got)


def test_embedding_ids_outside_the_table_and_shapes():
    w = torch.randn(10, 16, device=dev)
    ids = torch.tensor([[3, -1, 10], [9, 0, 2 ** 40]], device=dev)
    y = K().embedding(ids, w, scale=2.0)
    bad = torch.tensor([[False, True, True], [False, False, True]], device=dev)
    assert y.shape == (2, 3, 16) and torch.isnan(y[bad]).all() and torch.equal(y[~bad], 2 * w[ids[~bad]])
    dy = torch.randn(2, 3, 16, device=dev)
    dw = K().embedding_bwd(dy, ids, 10)
    want = torch.zeros(10, 16, device=dev)
    for (a, b) in ((0, 0), (1, 0), (1, 1)):
        want[ids[a, b]] = dy[a, b]
    assert torch.equal(dw, want)
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    assert K().embedding(none, w).shape == (0, 16)
    assert torch.equal(K().embedding_bwd(torch.zeros(0, 16, device=dev), none, 10), torch.zeros(10, 16, device=dev))
    wide = torch.randn(10, 40, device=dev)[:, 5:21]           # rows of a wider table, not aligned
    assert torch.equal(K().embedding(ids[1:, :2], wide), wide[ids[1:, :2]])


@pytest.mark.parametrize("N,V,C", [(300001, 1000, 8), (270000, (1 << 18) + 5, 5), (9000, 600000, 3), (5000, 1 << 19, 16), (100, 1 << 21, 2)])
def test_embedding_of_many_tokens_and_wide_tables(N, V, C):
    """More than 2^18 tokens (more places a workgroup), ids of 19 and 20 bits (three passes of the sort)."""
    test_embedding(N, V, C, ("f32", "f32", "f32"))


def test_padding_idx_outside_the_table_is_refused():
    from lrce import _native as N, ops  # noqa: F401  (registers the ops)
    w, ids = torch.randn(10, 16, device=dev, requires_grad=True), torch.tensor([3, 9, 0], device=dev)
    for pad in (-2, -10, 10):
        for call in (lambda: K().embedding_bwd(w.detach()[:3], ids, 10, padding_idx=pad), lambda: torch.ops.lrce.embedding(ids, w, 1.0, pad),
                     lambda: K().embedding_bwd(w.detach()[:3], ids, 10, padding_idx=pad, dw=torch.zeros(10, 16, device=dev))):
            with pytest.raises(N.NativeError, match="padding_idx"):
                call()
    torch.ops.lrce.embedding(ids, w, 1.0, 9).sum().backward()
    assert (w.grad[9] == 0).all() and (w.grad[[0, 3]] == 1).all()
