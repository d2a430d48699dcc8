"""Rotary positions and the cache write on a B200, against the formula in 64
bits.

Tolerance. The kernel forms the angle in 64 bits, reduces it to turns in fp32
(half a step of 2^-24 of at most half a turn, and as much again from doubling
into sincospif's argument: 2 pi * 2^-25 = 1.9e-7 rad) and takes sincospif
(2 ulp: 2.4e-7); with three fp32 roundings of values up to m (|a| + |b|) the
result before rounding is within 1e-6 * m * (|a| + |b|), and its rounding to
the type adds half a step, eps / 2 relative.
"""

import pytest
import torch

HD_CASES = [  # tokens, heads, kv_heads, hd, rot
    (1, 1, 1, 64, 64), (3, 16, 4, 64, 32), (37, 5, 1, 128, 128), (130, 32, 8, 128, 128), (19, 3, 3, 64, 26),
    (11, 7, 2, 128, 2), (5, 2, 1, 6, 4), (260, 4, 2, 80, 40), (9, 1, 70, 256, 256), (1030, 8, 8, 64, 8),
]


def turned(x, positions, freqs, interleaved, m):
    """The formula in 64 bits; also the magnitude |a| + |b| of each pair."""
    rot = 2 * freqs.numel()
    y = x.double().clone()
    mag = torch.zeros_like(y)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    t = (positions.double()[:, None] * freqs.double())[:, None]
    xa, xb = x.double()[..., a], x.double()[..., b]
    y[..., a] = m * (xa * t.cos() - xb * t.sin())
    y[..., b] = m * (xa * t.sin() + xb * t.cos())
    mag[..., a] = mag[..., b] = abs(m) * (xa.abs() + xb.abs())
    return y, mag


def near(got, want, mag):
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).tiny * eps  # a subnormal result rounds by half of this at most
    bound = want.abs() * (eps / 2) + 1e-6 * mag * (1 + eps) + tiny
    assert ((got.double() - want).abs() <= bound).all()


@pytest.fixture(scope="module")
def K():
    from transformer_optimization_b200 import _abi, kernels
    _abi.load()
    yield kernels
    assert _abi.device_status() == 0


def inputs(t, h, g, hd, rot, dtype, far, packed=True):
    from transformer_optimization_b200 import kernels
    gen = torch.Generator().manual_seed(t * 131 + h * 17 + hd + rot)
    qkv = torch.randn(t, h + 2 * g, hd, generator=gen).to(dtype).cuda()
    pos = torch.randint(-far, far, (t,), generator=gen).cuda()
    freqs, _ = kernels.rotary_freqs(rot, device="cuda")
    q, k, v = qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:]
    if not packed:
        q, k, v = (x.contiguous() for x in (q, k, v))
    return q, k, v, pos, freqs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,h,g,hd,rot", HD_CASES)
def test_rotary(K, t, h, g, hd, rot, interleaved, dtype):
    q, k, _, pos, freqs = inputs(t, h, g, hd, rot, dtype, 1000000)
    q0, k0 = q.clone(), k.clone()
    qo, ko = K.rotary(q, k, pos, freqs, interleaved=interleaved, mscale=1.25)
    near(qo, *turned(q, pos, freqs, interleaved, 1.25))
    near(ko, *turned(k, pos, freqs, interleaved, 1.25))
    assert torch.equal(q, q0) and torch.equal(k, k0)
    # in place, and queries alone: the same bits
    K.rotary(q, k, pos, freqs, interleaved=interleaved, mscale=1.25, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    alone, none = K.rotary(q0, None, pos, freqs, interleaved=interleaved, mscale=1.25)
    assert none is None and torch.equal(alone, qo)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_rotary_alignment(K, shift):
    """Bases and strides that rule out 16-byte accesses give the same bits."""
    q, k, _, pos, freqs = inputs(33, 4, 2, 64, 32, torch.float16, 5000, packed=False)
    want = K.rotary(q, k, pos, freqs)
    pad = torch.zeros(33, 6, 64 + shift, dtype=q.dtype, device="cuda")
    flat = torch.zeros(33 * 6 * 64 + shift, dtype=q.dtype, device="cuda")[shift:].view(33, 6, 64)
    for buf in (pad[..., shift:], flat):
        buf[:, :4], buf[:, 4:] = q, k
        got = K.rotary(buf[:, :4], buf[:, 4:], pos, freqs)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_rotary_special_values(K):
    """Infinities and NaN stay in their own pair; other pairs are unaffected."""
    q, _, _, pos, freqs = inputs(8, 2, 1, 64, 64, torch.float16, 100)
    want, _ = K.rotary(q, None, pos, freqs)
    bad = q.clone()
    bad[3, 1, 5], bad[4, 0, 40] = float("nan"), float("inf")
    got, _ = K.rotary(bad, None, pos, freqs)
    touched = torch.zeros_like(want, dtype=torch.bool)
    touched[3, 1, [5, 37]] = touched[4, 0, [8, 40]] = True
    assert torch.equal(got[~touched], want[~touched]) and not got[touched].isfinite().any()


@pytest.mark.gpu
def test_rotary_transpose_is_gradient(K):
    """<R x, y> = <x, R^T y> with R^T = rotary at -positions: the gradient of
    f(x) = <R x, y>, against differences of f along a direction d. f is linear
    in x, so the difference is exact but for the roundings of the kernel's
    outputs, eps / 2 of each term, and of the gradient's."""
    dt = torch.float16
    q, _, _, pos, freqs = inputs(40, 4, 1, 64, 48, dt, 3000)
    gen = torch.Generator().manual_seed(1)
    y, d = (torch.randn(q.shape, generator=gen).to(dt).cuda() for _ in range(2))
    grad, _ = K.rotary(y, None, -pos, freqs)
    x1 = (q.double() + d.double()).to(dt)
    step = x1.double() - q.double()
    r1, _ = K.rotary(x1, None, pos, freqs)
    r0, _ = K.rotary(q, None, pos, freqs)
    diff = ((r1.double() - r0.double()) * y.double()).sum()
    want = (grad.double() * step).sum()
    half = torch.finfo(dt).eps / 2

    def err(x, r, at):  # of one rotated tensor, per element
        return half * r.double().abs() + 1.1e-6 * turned(x, at, freqs, False, 1.0)[1]

    bound = ((err(x1, r1, pos) + err(q, r0, pos)) * y.double().abs()).sum() + (err(y, grad, -pos) * step.abs()).sum()
    assert (diff - want).abs() <= bound
    near(grad, *turned(y, -pos, freqs, False, 1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("swapped", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_append(K, page, swapped, interleaved, dtype):
    t, h, g, hd = 101, 6, 3, 64
    q, k, v, pos, freqs = inputs(t, h, g, hd, 32, dtype, 9000)
    pages = -(-t // page) + 4
    shape = (pages, g, page, hd) if swapped else (pages, page, g, hd)
    caches = [torch.full(shape, 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    kc, vc = (c.transpose(1, 2) if swapped else c for c in caches)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(page))[:t].cuda()
    slots[5], slots[77] = -1, -100  # padding tokens
    want_k, want_v = kc.clone(), vc.clone()
    qo, ko = K.rotary(q, k, pos, freqs, interleaved=interleaved)
    keep = slots >= 0
    want_k[slots[keep] // page, slots[keep] % page] = ko[keep]
    want_v[slots[keep] // page, slots[keep] % page] = v[keep]
    got = K.rotary_append(q, k, v, pos, freqs, kc, vc, slots, interleaved=interleaved)
    assert torch.equal(got, qo) and torch.equal(kc, want_k) and torch.equal(vc, want_v)


@pytest.mark.gpu
def test_rotary_append_past_the_cache():
    """A slot past the cache writes nothing and is reported."""
    from transformer_optimization_b200 import _abi, kernels as K
    q, k, v, pos, freqs = inputs(4, 2, 1, 64, 64, torch.float16, 10)
    kc, vc = (torch.zeros(2, 16, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    K.rotary_append(q, k, v, pos, freqs, kc, vc, torch.tensor([3, 32, 1 << 40, -1], device="cuda"))
    assert _abi.device_status() == 108 and _abi.device_status() == 0
    assert kc.flatten(0, 1).any(-1).nonzero().tolist() == [[3, 0]]
    assert vc.flatten(0, 1).any(-1).nonzero().tolist() == [[3, 0]]


@pytest.mark.gpu
def test_rotary_empty_stream_and_graph(K):
    q, k, _, pos, freqs = inputs(0, 2, 1, 64, 64, torch.float16, 10)
    qo, ko = K.rotary(q, k, pos, freqs)
    assert qo.shape == q.shape and ko.shape == k.shape
    q, k, _, pos, freqs = inputs(50, 2, 1, 64, 64, torch.float16, 10)
    want = K.rotary(q, k, pos, freqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.rotary(q, k, pos, freqs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = K.rotary(q, k, pos, freqs)
    q.neg_()
    g.replay()
    assert torch.equal(got[0], -want[0]) and torch.equal(got[1], want[1])


# ----------------------------------------------------------------- refusals (any host)
def _cpu(t=4, h=2, g=1, hd=64):
    z = torch.zeros
    return dict(q=z(t, h, hd).half(), k=z(t, g, hd).half(), v=z(t, g, hd).half(), positions=z(t, dtype=torch.int64),
                freqs=z(16, dtype=torch.float64), k_cache=z(2, 16, g, hd).half(), v_cache=z(2, 16, g, hd).half(),
                slots=z(t, dtype=torch.int64))


@pytest.mark.parametrize("name,value,match", [
    ("q", torch.zeros(4, 2, 64), "fp16 or bf16"),
    ("q", torch.zeros(4, 128).half(), "tokens, heads"),
    ("q", torch.zeros(4, 2, 128).half()[..., ::2], "unit inner"),
    ("k", torch.zeros(4, 1, 64).bfloat16(), "float16"),
    ("k", torch.zeros(5, 1, 64).half(), "same tokens"),
    ("v", torch.zeros(4, 2, 64).half(), "k's shape"),
    ("positions", torch.zeros(4, dtype=torch.int32), "int64"),
    ("positions", torch.zeros(5, dtype=torch.int64), "4 entries"),
    ("freqs", torch.zeros(16), "float64"),
    ("freqs", torch.zeros(33, dtype=torch.float64), "head of 64"),
    ("freqs", torch.zeros(0, dtype=torch.float64), "head of 64"),
    ("k_cache", torch.zeros(2, 16, 1, 32).half(), "k_cache"),
    ("v_cache", torch.zeros(3, 16, 1, 64).half(), "matching"),
    ("slots", torch.zeros(4, dtype=torch.int32), "int64"),
    ("q_out", torch.zeros(4, 1, 64).half(), "shape"),
])
def test_rotary_append_refuses(name, value, match):
    from transformer_optimization_b200 import kernels as K
    args = _cpu()
    args[name] = value
    with pytest.raises(ValueError, match=match):
        K.rotary_append(**args)


def test_rotary_refuses_cpu_and_bad_scaling():
    from transformer_optimization_b200 import kernels as K
    a = _cpu()
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rotary(a["q"], a["k"], a["positions"], a["freqs"])
    with pytest.raises(RuntimeError, match="CUDA"):
        K.rotary_append(**a)
    for bad in (dict(rot=3), dict(rot=0), dict(rot=8, scaling="other"), dict(rot=8, factor=0.5), dict(rot=8, base=0)):
        with pytest.raises(ValueError):
            K.rotary_freqs(**bad)


def test_rotary_abi_refuses_without_device():
    """The C entry refuses malformed arguments with a status, device or not."""
    from transformer_optimization_b200 import _abi
    lib = _abi.load()
    ok = [64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 64, 4, 2, 1, 64, 32, 1.0, 0, None]
    for at, value, code in [(0, None, 1), (3, None, 1), (6, None, 1), (9, None, 1), (12, None, 1), (13, None, 1),
                            (14, -1, 1), (15, -1, 1), (15, 1 << 40, 1), (17, 257, 1), (18, 33, 1), (18, 66, 1),
                            (19, float("inf"), 1), (20, 8, 1), (0, 65, 2), (12, 4, 2)]:
        args = list(ok)
        args[at] = value
        assert lib.tf_rotary(*args) == code, (at, value)
        assert lib.tf_last_error()


@pytest.mark.parametrize("at,value", [(4, 0), (4, 64), (5, 0), (5, 62), (10, 32), (11, 0)])
def test_rotary_abi_refuses_overlapping_results(at, value):
    """Rows of an output in one place would be written in any order; inputs may repeat (stride 0)."""
    from transformer_optimization_b200 import _abi
    lib = _abi.load()
    args = [64, 0, 0, 64, 128, 64, 64, 0, 0, 64, 128, 64, 64, 64, 4, 2, 2, 64, 32, 1.0, 0, None]
    args[at] = value
    assert lib.tf_rotary(*args) == 1
    assert b"overlap" in lib.tf_last_error()


@pytest.mark.parametrize("at,value", [(16, 0), (16, 1024), (17, 64), (18, 0)])
def test_rotary_append_abi_refuses_overlapping_cache(at, value):
    from transformer_optimization_b200 import _abi
    lib = _abi.load()
    args = [64, 128, 64, 64, 128, 64, 64, 128, 64, 64, 128, 64, 64, 64, 64, 64, 2048, 128, 64, 3, 16, 64, 4, 2, 2, 64, 32,
            1.0, 0, None]
    args[at] = value
    assert lib.tf_rotary_append(*args) == 1
    assert b"overlap" in lib.tf_last_error()


def test_rotary_freqs_scaling():
    from transformer_optimization_b200 import kernels as K
    f, m = K.rotary_freqs(64)
    assert m == 1.0 and f.dtype == torch.float64 and f[0] == 1.0
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64))
    assert torch.allclose(K.rotary_freqs(64, scaling="linear", factor=4.0)[0], f / 4, rtol=1e-15)
    ntk, _ = K.rotary_freqs(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and abs(ntk[-1] / (f[-1] / 4) - 1) < 1e-12
    parts, m = K.rotary_freqs(64, scaling="parts", factor=4.0)
    assert m > 1.1 and parts[0] == f[0] and abs(parts[-1] / (f[-1] / 4) - 1) < 1e-12
    assert ((parts <= f) & (parts >= f / 4 * (1 - 1e-15))).all()
