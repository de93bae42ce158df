"""Attention at general lengths (csrc/attention.hip, attention_bwd.hip; lrce.kernels.attention / attention_bwd) against the
64-bit reference of attention_ref.py, every output and gradient within its derived allowance."""
import pytest
import torch

from attention_ref import check, reference

pytestmark = pytest.mark.gpu
dev = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def K():
    from lrce import kernels
    return kernels


def make(B, Lq, Lk, H, Hk, D, dtype, seed=0, mask=None, packed=False, spread=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g, device=dev) * spread).to(DT[dtype])
    if packed:
        q, k, v = r(B, Lq, H + 2 * Hk, D).split([H, Hk, Hk], 2)
    else:
        q, k, v = r(B, Lq, H, D), r(B, Lk, Hk, D), r(B, Lk, Hk, D)
    do = r(B, Lq, H, D)
    m = None
    if mask == "tail":
        n = torch.tensor([max(1, Lk - 5 * b * Lk // 7 % Lk) for b in range(B)], device=dev)
        m = torch.arange(Lk, device=dev)[None] < n[:, None]
    elif mask == "random":
        m = torch.rand(B, Lk, generator=g, device=dev) < 0.6
        m[0] = False                                                  # a batch row that sees nothing
    elif mask == "blocks":                                            # whole tiles hidden, also the first
        m = (torch.arange(Lk, device=dev)[None] // 64 + torch.arange(B, device=dev)[:, None]) % 3 == 1
    return q, k, v, do, m


def run(q, k, v, do, m, causal=False, scale=None, backward=True, what=""):
    out, lse = K().attention(q, k, v, key_mask=m, causal=causal, scale=scale)
    got = {"out": out, "lse": lse}
    if backward:
        got["dq"], got["dk"], got["dv"] = K().attention_bwd(do, q, k, v, out, lse, key_mask=m, causal=causal, scale=scale)
    torch.cuda.synchronize()
    check(got, reference(q, k, v, m, causal, scale, do if backward else None), what)
    return got


SHAPES = [
    # B, Lq, Lk, H, Hk
    (1, 1, 1, 1, 1), (2, 1, 33, 4, 2), (3, 31, 31, 2, 2), (2, 64, 65, 3, 1), (2, 129, 127, 4, 4), (1, 257, 300, 4, 1), (2, 100, 700, 6, 2),
]


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_backward(shape, D, dtype):
    B, Lq, Lk, H, Hk = shape
    for causal in (False, True):
        for mask in (None, "random"):
            run(*make(B, Lq, Lk, H, Hk, D, dtype, seed=Lq + Lk, mask=mask), causal=causal, what=f"causal={causal} mask={mask}")


@pytest.mark.parametrize("mask", ["tail", "blocks", "random"])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64)])
def test_masks(mask, dtype, D):
    for mt in (torch.bool, torch.uint8, torch.int32, torch.int64):
        q, k, v, do, m = make(4, 150, 450, 4, 2, D, dtype, seed=7, mask=mask)
        run(q, k, v, do, m.to(mt) * (3 if mt != torch.bool else 1), what=str(mt))


@pytest.mark.parametrize("D", [32, 96, 128])
def test_single_tokens_over_a_long_axis(D):
    """Few rows: the keys are split over waves and workgroups and joined (one and several workgroups, several row tiles)."""
    for B, Lq, Lk, H, Hk, causal, mask in ((1, 1, 20000, 8, 1, False, None), (3, 1, 9001, 10, 2, False, "random"), (2, 5, 3000, 8, 2, True, "tail"),
                                           (2, 1, 200, 4, 4, False, "blocks"), (1, 40, 4096, 2, 1, True, None), (40, 1, 1000, 24, 8, True, "tail")):
        run(*make(B, Lq, Lk, H, Hk, D, "bf16", seed=Lk, mask=mask), causal=causal, backward=False, what=f"{B} {Lq} {Lk} {H} {Hk}")
