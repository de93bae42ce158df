"""Attention in 64 bits and how far a kernel's outputs may be from it, element by element (test_attention_gpu.py).

The allowance counts what the computation cannot avoid: u = half a step of the 16-bit type where a weight or a result is
rounded to it, 2^-24 for each 32-bit operation on the way, propagated by the triangle inequality."""
import math

import torch

F64 = torch.float64
E32 = 2.0 ** -24


def allowed_pairs(B, Lq, Lk, key_mask, causal, device):
    ok = torch.ones(B, 1, Lq, Lk, dtype=torch.bool, device=device)
    if key_mask is not None:
        ok = ok & (key_mask != 0)[:, None, None, :]
    if causal:
        i = torch.arange(Lq, device=device)[:, None] + (Lk - Lq)
        ok = ok & (torch.arange(Lk, device=device)[None] <= i)
    return ok


def reference(q, k, v, key_mask=None, causal=False, scale=None, dout=None):
    """dict name -> (value f64, allowed error f64), laid out as the operator's outputs."""
    dt, dev = q.dtype, q.device
    u = torch.finfo(dt).eps / 2
    tiny = float(torch.finfo(dt).tiny) * torch.finfo(dt).eps          # smallest step of the type, near zero
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    ok = allowed_pairs(B, Lq, Lk, key_mask, causal, dev).expand(B, H, Lq, Lk)
    seen = (key_mask != 0)[:, :, None, None] if key_mask is not None else torch.ones(B, Lk, 1, 1, dtype=torch.bool, device=dev)
    Q = q.to(F64).transpose(1, 2)
    K = torch.where(seen, k.to(F64), 0.0).transpose(1, 2).repeat_interleave(G, 1)
    V = torch.where(seen, v.to(F64), 0.0).transpose(1, 2).repeat_interleave(G, 1)
    s = (scale * (Q @ K.transpose(-1, -2))).masked_fill(~ok, -math.inf)
    sa = scale * (Q.abs() @ K.abs().transpose(-1, -2))                # what the 32-bit sums are relative to
    m = s.amax(-1, keepdim=True) if Lk else torch.full((B, H, Lq, 1), -math.inf, dtype=F64, device=dev)
    mz = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(s - mz)
    l = e.sum(-1, keepdim=True)
    lz = torch.where(l == 0, 1.0, l)
    p = e / lz
    o = p @ V
    lse = torch.where(l > 0, mz + lz.log(), -math.inf)
    # relative error of a weight before it is rounded: the score's 32-bit sum, its scaling, the maximum's, the exponential's
    es = ((D + 4) * E32 * sa + 4 * E32 * (s.masked_fill(~ok, 0.0).abs() + mz.abs()) + 4 * E32).masked_fill(~ok, 0.0)
    emax = es.amax(-1, keepdim=True) if Lk else torch.zeros_like(m)
    sums = (Lk + 8) * E32                                             # of sums over the keys
    pv = p @ V.abs()
    # a weight below the type's normal range is off by its smallest step; weights are relative to a maximum of at least 1
    floor = tiny * (ok.to(F64) @ V.abs()) / lz
    eo = 1.01 * (u * o.abs() + (u + 2 * emax + 2 * sums) * pv + floor) + tiny
    out = {"out": (o.transpose(1, 2), eo.transpose(1, 2)),
           "lse": (lse[..., 0], (emax + sums + 4 * E32 * (1 + mz.abs() + lz.log().abs()))[..., 0])}
    if dout is None:
        return out
    d = dout.to(F64).transpose(1, 2)
    dp = d @ V.transpose(-1, -2)
    delta = (d * o).sum(-1, keepdim=True)
    # the backward recomputes the weights from the rounded lse and forms delta from the rounded out
    ep = es + (emax + sums + 8 * E32 * (1 + mz.abs() + lz.log().abs()))
    edp = (D + 2) * E32 * (d.abs() @ V.abs().transpose(-1, -2)) + (d.abs() * eo).sum(-1, keepdim=True) + (D + 2) * E32 * (d * o).abs().sum(-1, keepdim=True)
    ds = p * (dp - delta)
    eds = (u + ep + 4 * E32) * ds.abs() + p * (1 + u + ep) * edp + tiny
    qsum = (Lq * G + 8) * E32

    def heads(t):                                                     # sum over the query heads of a key head
        return t.view(B, Hk, G, Lk, D).sum(2)

    dq = scale * (ds @ K)
    dk = heads(scale * (ds.transpose(-1, -2) @ Q))
    dv = heads(p.transpose(-1, -2) @ d)
    edq = scale * ((eds + sums * ds.abs()) @ K.abs())
    edk = heads(scale * ((eds + qsum * ds.abs()).transpose(-1, -2) @ Q.abs()))
    edv = heads((((u + ep + qsum) * p) + tiny * ok).transpose(-1, -2) @ d.abs())
    for name, x, ex in (("dq", dq, edq), ("dk", dk, edk), ("dv", dv, edv)):
        out[name] = (x.transpose(1, 2), (1.01 * (ex + (u + 4 * E32) * x.abs()) + tiny).transpose(1, 2))
    return out


def check(got, want, what=""):
    """got: dict of tensors; each element within its allowance, infinities equal, no NaN."""
    for name, t in got.items():
        x, e = want[name]
        t = t.to(F64)
        assert t.shape == x.shape, (what, name, t.shape, x.shape)
        if t.numel() == 0:
            continue
        same = t == x                                                 # covers equal infinities
        off = torch.where(same, 0.0, (t - x).abs())
        bad = ~(off <= e)
        worst = torch.where(same, 0.0, off / e).nan_to_num(nan=math.inf).max().item()
        assert not bad.any(), f"{what} {name}: {int(bad.sum())} of {bad.numel()} values off, worst {worst:.3g} of the allowance"
