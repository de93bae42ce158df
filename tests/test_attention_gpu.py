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


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_many_rows_over_many_keys(D, dtype):
    """Enough row tiles that a workgroup's waves take rows of their own, over several key tiles."""
    for Lq, Lk, causal, mask in ((401, 500, False, None), (401, 500, True, "tail"), (500, 401, True, None), (416, 321, False, "blocks"),
                                 (385, 192, True, "random")):
        run(*make(3, Lq, Lk, 24, 6, D, dtype, seed=Lq, mask=mask), causal=causal, what=f"{Lq} {Lk} {causal} {mask}")


@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_middling_rows_over_many_keys(D):
    """256 to 768 row tiles: the waves of a workgroup divide the keys."""
    for B, Lq, Lk, H, Hk, causal, mask in ((4, 257, 613, 8, 8, False, None), (5, 250, 700, 12, 4, True, "tail"), (4, 333, 449, 10, 5, False, "random"),
                                           (6, 200, 192, 8, 2, True, "blocks")):
        run(*make(B, Lq, Lk, H, Hk, D, "bf16", seed=Lq, mask=mask), causal=causal, what=f"{B} {Lq} {Lk} {H} {Hk}")


@pytest.mark.parametrize("D", [64, 96])
def test_masks_longer_than_a_workgroup_reads_at_once(D):
    """The mask's words are read 4096 keys (keys divided over the waves) or 16384 keys (rows divided) at a time."""
    run(*make(64, 1, 4500, 8, 8, D, "bf16", seed=1, mask="tail"), what="a workgroup for each cache")
    run(*make(70, 3, 4200, 8, 8, D, "bf16", seed=2, mask="random"), causal=True, what="a workgroup for each cache, causal")


@pytest.mark.parametrize("mask,causal", [("random", False), ("tail", True)])
def test_masks_longer_than_16384_keys(mask, causal):
    run(*make(2, 820, 16500, 16, 2, 32, "bf16", seed=3, mask=mask), causal=causal)


def test_backward_of_single_tokens_over_long_caches():
    for B, Lq, Lk, H, Hk, D, causal, mask in ((2, 1, 9001, 8, 2, 128, False, "tail"), (1, 1, 20000, 4, 4, 64, True, None), (3, 2, 5000, 12, 3, 96, True, "random")):
        run(*make(B, Lq, Lk, H, Hk, D, "bf16", seed=Lk, mask=mask), causal=causal, what=f"{B} {Lq} {Lk} {H} {Hk}")


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_short_axes(D, dtype):
    """Up to 64 queries and keys, whose gradients one launch forms: shared heads, masks, rows before the first key."""
    for B, Lq, Lk, H, Hk in ((2, 64, 64, 8, 2), (1, 33, 64, 8, 1), (3, 64, 31, 6, 6), (4, 1, 1, 2, 1), (520, 3, 5, 10, 1), (2, 40, 57, 18, 2)):
        for causal, mask in ((False, None), (True, None), (False, "random"), (True, "tail")):
            run(*make(B, Lq, Lk, H, Hk, D, dtype, seed=Lq, mask=mask), causal=causal, scale=0.3, what=f"{B} {Lq} {Lk} {H} {Hk} {causal} {mask}")


def test_few_shares_or_many_rows_over_long_axes():
    """Where one-wave shares would be few, or their join long, a workgroup's waves have the keys between them; one case each side."""
    for B, Lq, Lk, H, Hk, D, causal, mask in ((7, 1100, 1100, 1, 1, 32, True, "tail"), (1, 1, 1100, 8, 1, 64, False, None), (1, 1, 3200, 8, 1, 64, True, None),
                                              (4, 1, 2000, 12, 12, 64, False, "random"), (2, 33, 3000, 8, 2, 128, True, "blocks"), (1, 200, 4000, 8, 8, 96, True, None)):
        run(*make(B, Lq, Lk, H, Hk, D, "bf16", seed=Lk, mask=mask), causal=causal, what=f"{B} {Lq} {Lk} {H} {Hk} {D}")


def test_one_row_over_more_than_256_shares():
    """The join takes 256 shares at a time; some of them, the first among them, see nothing."""
    Lk, H, D = 200001, 2, 32
    assert K()._attn_ws(False, 1, H, 1, 1, Lk, D) > 256 * H * (D + 2)
    q, k, v, do, _ = make(1, 1, Lk, H, 1, D, "bf16", seed=11)
    m = torch.rand(1, Lk, generator=torch.Generator(device=dev).manual_seed(12), device=dev) < 0.4
    for a, b in ((0, 1500), (60000, 63000), (150000, 199990)):
        m[:, a:b] = False
    for mask in (m, None):
        run(q, k, v, do, mask, what=f"mask={mask is not None}")
