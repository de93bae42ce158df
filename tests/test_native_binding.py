"""The host side of the attention, norm + rotation and embedding calls: the module built from csrc/binding.cpp and the Python path
launch the same, and what the module does not take (other layouts, wrong arguments) the Python path does or refuses."""
import pytest
import torch

from lrce import _native as N
from lrce import kernels as K

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def test_the_module_takes_nothing_from_the_host():
    """CPU tensors, wrong counts and things that are no tensors: None, never an error or a launch."""
    b = N.binding()
    q = torch.zeros(1, 4, 2, 64, dtype=BF)
    w, p, f, ids, t = torch.ones(64), torch.arange(4), torch.ones(32), torch.zeros(3, dtype=torch.long), torch.zeros(5, 8)
    assert b.attention(q, q, q, None, False, None, 0, 0) is None
    assert b.attention_bwd(q, q, q, None, False, None, q, q, w, 0, 0) is None
    assert b.qk_norm_rope(q, q, w, w, p, f, 1e-6, False, 0, 0) is None
    assert b.qk_norm_rope_bwd(q, q, w, w, p, f, 1e-6, False, q, q, 0, 0) is None
    assert b.embedding(ids, t, 1.0, None, 0, 0) is None
    assert b.embedding_bwd(t, ids, 5, 1.0, -1, 0, 0) is None
    for f in (b.attention, b.attention_bwd, b.qk_norm_rope, b.qk_norm_rope_bwd, b.embedding, b.embedding_bwd):
        assert f() is None
        assert f(*[None] * 8) is None and f(*["x"] * 12) is None
    with pytest.raises(TypeError):
        b.bind(1)
    with pytest.raises(ValueError):
        b.bind(*[0] * 10)


def test_the_module_is_built_for_torchs_abi(tmp_path):
    """The compile line has the loading interpreter's torch and its C++ ABI, not the compiler's default."""
    import os
    import subprocess
    import sys
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(N.__file__)))), "csrc")
    out = str(tmp_path / "b.so")
    line = subprocess.run(["make", "-s", "-C", csrc, "-B", "CXX=echo", "PYTHON=" + sys.executable, "BINDING=" + out, out], check=True,
                          capture_output=True, text=True).stdout
    assert f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())} " in line and f"-I{os.path.dirname(torch.__file__)}/include" in line


def gpu(seed, *shape, dtype=BF):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def through_python(monkeypatch, f):
    with monkeypatch.context() as m:
        m.setattr(K, "_direct", lambda t: (None, 0, 0))
        return f()


def same(monkeypatch, f):
    a, b = f(), through_python(monkeypatch, f)
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and x.device == y.device and not x.requires_grad
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())


def here():
    dev = torch.cuda.current_device()
    return dev, torch.cuda.current_stream().cuda_stream


@pytest.mark.gpu
@pytest.mark.parametrize("B,Lq,Lk,H,Hk,D,dtype,mask,causal,scale", [
    (2, 40, 40, 4, 4, 64, F16, torch.bool, False, None), (3, 1, 700, 8, 2, 128, BF, torch.int64, False, 0.2),
    (1, 1, 9000, 4, 1, 96, BF, None, True, None), (2, 300, 333, 4, 2, 32, BF, torch.int32, True, 1),
    (2, 0, 5, 2, 1, 64, BF, None, False, None), (2, 5, 0, 2, 1, 64, BF, None, True, None)])
def test_attention_is_the_same_both_ways(monkeypatch, B, Lq, Lk, H, Hk, D, dtype, mask, causal, scale):
    q, k, v = gpu(1, B, H, Lq, D, dtype=dtype).transpose(1, 2), gpu(2, B, Lk, Hk, D, dtype=dtype), gpu(3, B, Lk, 2, Hk, D, dtype=dtype)[:, :, 1]
    g = gpu(4, B, Lq, H, D, dtype=dtype).requires_grad_()
    m = None if mask is None else (gpu(5, B, 2 * Lk, dtype=F32) > 0).to(mask)[:, :Lk]
    out, lse = K.attention(q, k, v, m, causal, scale)
    assert N.binding().attention(q, k, v, m, causal, scale, *here()) is not None
    assert N.binding().attention_bwd(q, k, v, m, causal, scale, g, out, lse, *here()) is not None
    same(monkeypatch, lambda: K.attention(q, k, v, m, causal, scale))
    same(monkeypatch, lambda: K.attention_bwd(g, q, k, v, out, lse, m, causal, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("D,R,inter,two", [(64, 64, False, True), (96, 32, True, False), (8, 2, True, True), (256, 200, False, False)])
def test_norm_and_rotation_are_the_same_both_ways(monkeypatch, dtype, D, R, inter, two):
    B, L, H, Hk = 2, 37, 4, 2
    q, k, w1, w2 = gpu(1, B, L, H, D, dtype=dtype), gpu(2, B, Hk, L, D, dtype=dtype).transpose(1, 2), gpu(3, D, dtype=F32), gpu(4, D, dtype=F32)
    f = gpu(5, R // 2, dtype=F32).abs()
    pos = torch.arange(L, device="cuda")
    pos = torch.stack([pos, pos + 7]).int() if two else pos
    gq, gk = gpu(6, B, L, H, D, dtype=dtype), gpu(7, B, L, Hk, D, dtype=dtype)
    assert N.binding().qk_norm_rope(q, k, w1, w2, pos, f, 1e-6, inter, *here()) is not None
    assert N.binding().qk_norm_rope_bwd(q, k, w1, w2, pos, f, 1e-6, inter, gq, gk, *here()) is not None
    same(monkeypatch, lambda: K.qk_norm_rope(q, k, w1, w2, pos, f, 1e-5, inter))
    same(monkeypatch, lambda: K.qk_norm_rope_bwd(gq, gk, q, k, w1, w2, pos, f, 1e-5, inter))


@pytest.mark.gpu
@pytest.mark.parametrize("wt,yt", [(F32, None), (F32, BF), (BF, BF), (F16, None)])
@pytest.mark.parametrize("shape", [(), (0,), (33,), (3, 700)])
def test_embedding_is_the_same_both_ways(monkeypatch, wt, yt, shape):
    w = gpu(1, 50, 24, dtype=wt).requires_grad_()
    ids = torch.randint(-1, 51, shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.int32 if len(shape) > 1 else torch.int64)
    dy = gpu(3, *shape, 24, dtype=yt or wt)
    assert N.binding().embedding(ids, w, 2.5, yt, *here()) is not None and N.binding().embedding_bwd(dy, ids, 50, 2.5, 3, *here()) is not None
    same(monkeypatch, lambda: K.embedding(ids, w, 2.5, yt))
    same(monkeypatch, lambda: K.embedding_bwd(dy, ids, 50, 2.5, 3))


@pytest.mark.gpu
def test_what_the_module_does_not_take():
    """None from the module, and a refusal (not a launch) from the call."""
    q, k = gpu(1, 2, 8, 4, 64), gpu(2, 2, 9, 2, 64)
    w, pos, f = gpu(3, 64, dtype=F32), torch.arange(8, device="cuda"), gpu(4, 32, dtype=F32)
    b = N.binding()
    mask = torch.ones(2, 9, dtype=torch.bool, device="cuda")
    for args in [(q, k, k[:, :8]), (q, k[:1], k[:1]), (q, k.half(), k), (q[..., :48], k[..., :48], k[..., :48]), (q[:, :, :3], k, k), (q[0], k, k),
                 (q, k.cpu(), k), (q, k, k, mask[:, :8]), (q, k, k, mask.float()), (q, k, k, mask.cpu()), (q, k, k, None, False, 0.0),
                 (q, k, k, None, False, -1.0), (q, k, k, None, False, float("nan"))]:
        full = args + (None, False, None)[len(args) - 3:]
        assert b.attention(*full, *here()) is None
        with pytest.raises(N.NativeError):
            K.attention(*args)
    for args in [(q, q, w[:32], w, pos, f), (q, q, w.half(), w, pos, f), (q, q, w, w, pos[:7], f), (q, q, w, w, pos.float(), f), (q, q, w, w, pos, w),
                 (q, q[:, :7], w, w, pos, f), (q, q, w, w, pos, f, -1.0), (q[..., :12], q[..., :12], w[:12], w[:12], pos, f[:6])]:
        full = args + (1e-6, False)[len(args) - 6:]
        assert b.qk_norm_rope(*full, *here()) is None
        with pytest.raises(N.NativeError):
            K.qk_norm_rope(*args)
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    for args in [(ids.float(), w[None], 1.0, None), (ids, w, 1.0, None), (ids, w[None].bfloat16(), 1.0, F32), (ids.cpu(), w[None], 1.0, None)]:
        assert b.embedding(*args, *here()) is None
        with pytest.raises(N.NativeError):
            K.embedding(*args)
    # taken over by the Python path: a copy made there, or another stride
    dev, stream = here()
    odd = torch.empty(2 * 8 * 4 * 64 + 1, dtype=BF, device="cuda")[1:].view(2, 8, 4, 64).copy_(q)
    assert b.attention(odd, k, k, None, False, None, dev, stream) is None and torch.equal(K.attention(odd, k, k)[0], K.attention(q, k, k)[0])
    turned = w.view(2, 32).t()
    assert b.embedding(ids, turned, 1.0, None, dev, stream) is None and torch.equal(K.embedding(ids, turned), turned[ids])
    assert b.attention(q, k, k, None, False, None, dev + 1, stream) is None


@pytest.mark.gpu
def test_calls_from_several_threads_at_once():
    """Each thread on a stream of its own, through the module: short backward, divided keys, rotation, embedding."""
    import threading
    cases = [(2, 40, 40, 4, 2, 64), (1, 1, 5000, 8, 2, 128), (2, 300, 333, 4, 2, 32)]
    w, pos, f = torch.ones(64, device="cuda"), torch.arange(50, device="cuda"), torch.linspace(1, 0.01, 32, device="cuda")
    x, ids, tab = gpu(9, 2, 50, 4, 64), torch.arange(700, device="cuda") % 13, gpu(8, 20, 48, dtype=F32)

    def work(i):
        B, Lq, Lk, H, Hk, D = cases[i % 3]
        q, k, v = gpu(i, B, Lq, H, D), gpu(i + 10, B, Lk, Hk, D), gpu(i + 20, B, Lk, Hk, D)
        out, lse = K.attention(q, k, v)
        return [out, lse, *K.attention_bwd(q, q, k, v, out, lse), *K.qk_norm_rope(x, x, w, w, pos, f),
                *K.qk_norm_rope_bwd(x, x, x, x, w, w, pos, f), K.embedding(ids, tab), K.embedding_bwd(K.embedding(ids, tab), ids, 20)]
    want = [work(i) for i in range(6)]
    torch.cuda.synchronize()
    bad = []

    def thread(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = work(i)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
            s.synchronize()
    threads = [threading.Thread(target=thread, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
