"""Rotary positions and norms of queries and keys (`makani_b200/ops/rotary.py`) against their definition in 64 bits.

Tolerances, element by element.  An angle is reduced to a fraction of a turn in 64 bits and rounded to fp32 (2^-26 turns, 4e-7 of an angle with the two steps that
sine and cosine may be off): A = 2^-20 of the two values that are turned into one another, the products' roundings with it.  Sums over at most 256 channels, the
square root and the quotient are counted as F = 2^-18 of the sum of magnitudes.  A result is then rounded once, half a step of its type.

    xh off by F (|xh| + rstd mean|x|) =: e;   y = xh w + b off by e |w| + F |b|
    out off by A (|y| + |y'|) + (what y and y' are off)
    g = dout turned back, off by A (|dout| + |dout'|) =: d
    dx = rstd (g w - m0 - xh m1) off by rstd (d |w| + mean(d |w|) + 4 F (|g w| + mean|g w|) + (|xh| + e / F) (4 F mean|g w xh| + mean(d |w xh|)) + ...)
    dw = sum g xh off by sum (d |xh| + |g| e) + 2^-15 sum |g xh| (partial sums of at most some hundred rows one after the other)"""

import copy
import math
import pickle

import pytest
import torch

from makani_b200.ops import _ext
from makani_b200.ops import rotary as rot

A = 2.0 ** -20
F = 2.0 ** -18


def _partner(axes, D):
    at = torch.arange(D)
    sign = torch.zeros(D, dtype=torch.float64)
    start = 0
    for b in axes.bands if axes is not None else ():
        for i in range(b // 2):
            lo, hi = (start + 2 * i, start + 2 * i + 1) if axes.interleaved else (start + i, start + b // 2 + i)
            at[lo], at[hi], sign[lo], sign[hi] = hi, lo, -1.0, 1.0
        start += b
    return at, sign


def _angles(axes, positions, D):
    """[.., 1, D], fp64, from the formula."""
    out = torch.zeros(*positions.shape[:-1], D, dtype=torch.float64, device=positions.device)
    start = 0
    for a, (b, base) in enumerate(zip(axes.bands, axes.base)):
        for i in range(b // 2):
            turn = positions[..., a].double() * base ** (-2.0 * i / b)
            for c in ((start + 2 * i, start + 2 * i + 1) if axes.interleaved else (start + i, start + b // 2 + i)):
                out[..., c] = turn
        start += b
    return out[..., None, :]


def _oracle(x, w, b, positions, axes, eps, norm, do=None):
    """Results, and with `do` gradients (dx, dw, db), each with what it may be off before the last rounding."""
    x = x.detach().double()
    D = x.shape[-1]
    w64 = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    b64 = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    if norm is None:
        y, y_off = x, torch.zeros_like(x)
    else:
        mean = x.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(x[..., :1])
        rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
        xh = (x - mean) * rstd
        e = F * (xh.abs() + rstd * x.abs().mean(-1, keepdim=True))
        y, y_off = xh * w64 + b64, e * w64.abs() + F * b64.abs()
    if positions is None:
        cos, sin, at = torch.ones_like(x), torch.zeros_like(x), torch.arange(D, device=x.device)
    else:
        at, sign = (t.to(x.device) for t in _partner(axes, D))
        a = _angles(axes, positions, D)
        cos, sin = torch.cos(a) * torch.ones_like(x), torch.sin(a) * sign * torch.ones_like(x)
    alone = (sin == 0) if positions is None else (sign == 0).expand_as(x)
    mate = torch.where(alone, torch.zeros_like(y), y[..., at])
    out = cos * y + sin * mate
    off = A * (y.abs() + mate.abs()) + y_off + torch.where(alone, torch.zeros_like(y_off), y_off[..., at])
    if do is None:
        return (out, off), None
    do = do.double()
    mate = torch.where(alone, torch.zeros_like(do), do[..., at])
    g, d = cos * do - sin * mate, A * (do.abs() + mate.abs())
    if norm is None:
        return (out, off), ((g, d), None, None)
    gw, dw_ = g * w64, d * w64.abs()
    m = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    m0 = m(gw) if norm == "layer" else 0.0
    dx = rstd * (gw - m0 - xh * m(gw * xh))
    dx_off = rstd * (dw_ + m(dw_) + 4 * F * (gw.abs() + m(gw.abs())) + (xh.abs() + e / F) * (4 * F * m((gw * xh).abs()) + m(dw_ * xh.abs()) + m(gw.abs() * e))
                     + e * m((gw * xh).abs()))
    flat = lambda t: t.reshape(-1, D).sum(0)  # noqa: E731
    return (out, off), ((dx, dx_off), (flat(g * xh), flat(d * xh.abs() + g.abs() * e) + 2.0 ** -15 * flat((g * xh).abs())),
                        (flat(g), flat(d) + 2.0 ** -15 * flat(g.abs())))


def _close(got, want, off, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    diff = (got.double() - want).abs()
    bound = off * (1 + 2.0 ** -8) + torch.finfo(got.dtype).eps / 2 * want.abs() + 1e-30
    bad = ~(diff <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((diff / bound).nan_to_num(9e9)[bad].max()):.2f} of the bound"


def _check(q, k, axes, positions, norm, params, eps=1e-5, grads=True, seed=0):
    """Forward and backward of one call, every output."""
    g = torch.Generator(q.device).manual_seed(seed + 77)
    leaves = {"q": q, "k": k, **{n: p for n, p in params.items() if p is not None}}
    for t in leaves.values():
        t.requires_grad_(grads)
    if norm is None:
        out = rot.rotary_qk(q, k, positions, axes)
    else:
        out = rot.norm_rotary_qk(q, k, params.get("q_weight"), params.get("k_weight"), positions, axes, params.get("q_bias"), params.get("k_bias"), eps, norm)
    do = [torch.randn(t.shape, device=q.device, generator=g).to(t.dtype) for t in out]
    got = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), do))) if grads else {}
    for n, x, y, d in zip("qk", (q, k), out, do):
        (want, off), back = _oracle(x, params.get(n + "_weight"), params.get(n + "_bias"), positions, axes, eps, norm, d if grads else None)
        assert y.dtype == x.dtype and y.is_contiguous()
        _close(y.detach(), want, off, n)
        if grads:
            assert got[n].dtype == x.dtype
            _close(got[n], *back[0], "d" + n)
            for p, b in ((n + "_weight", back[1]), (n + "_bias", back[2])):
                if p in got:
                    assert got[p].dtype == leaves[p].dtype
                    _close(got[p], *b, "d" + p)
    return out, got


def _params(D, dev, g, bias=True, dtype=torch.float32):
    r = lambda: torch.randn(D, device=dev, generator=g).to(dtype)  # noqa: E731
    p = dict(q_weight=1 + 0.3 * r(), k_weight=1 + 0.3 * r())
    return {**p, "q_bias": 0.3 * r(), "k_bias": 0.3 * r()} if bias else p


def _grid(N, axes, dev):
    at = torch.arange(N, device=dev)
    return torch.stack([(at // 7 ** a) % 13 + 3 * a for a in range(axes)], -1).int()


# ---------------------------------------------------------------------------------------------------- any machine

def test_axes():
    a = rot.RotaryAxes((8, 4), base=(100.0, 10.0), interleaved=True)
    assert len(a) == 2 and a.channels == 12 and a.frequencies[0] == 1.0 and a.frequencies[5] == 10.0 ** -0.5
    assert a == copy.deepcopy(a) == pickle.loads(pickle.dumps(a)) and hash(a) == hash(copy.copy(a)) and a != rot.RotaryAxes((8, 4))
    for bad in ((), (3,), (0,), (2, 2, 2, 2, 2), (2.0,), (True,)):
        with pytest.raises(ValueError, match="bands"):
            rot.RotaryAxes(bad)
    for base in (0.0, -1.0, math.inf, (1.0,)):
        with pytest.raises(ValueError, match="base"):
            rot.RotaryAxes((2, 2), base=base)
    at = rot.grid_positions(2, 3, first=1)
    assert at.dtype == torch.int32 and at.tolist() == [[0, 0], [0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]
    with pytest.raises(ValueError):
        rot.grid_positions()


def test_refusals():
    x, axes, at = torch.randn(2, 5, 4, 8), rot.RotaryAxes((4, 4)), torch.zeros(5, 2)
    k, w = torch.randn(2, 5, 2, 8), torch.ones(8)
    for bad in (x[0, 0], x.long(), x[..., :0]):
        with pytest.raises(ValueError):
            rot.rotary(bad, at, axes)
    for bad in (at[:4], at[:, :1], at[None], at.half(), at.clone().requires_grad_(), at[None].expand(3, 5, 2)):
        with pytest.raises(ValueError, match="positions"):
            rot.rotary(x, bad, axes)
    with pytest.raises(ValueError, match="turn"):
        rot.rotary(x[..., :6], at, axes)
    with pytest.raises(ValueError, match="together"):
        rot.rotary(x, at, None)
    with pytest.raises(ValueError):
        rot.rotary(x, None, None)
    with pytest.raises(ValueError):
        rot.rotary_qk(x, k, None, None)
    for bad in (k[:1], k[:, :4], k[..., :4], k.double(), k[0]):
        with pytest.raises(ValueError, match="same tokens"):
            rot.rotary_qk(x, bad, at, axes)
    with pytest.raises(ValueError, match="norm"):
        rot.norm_rotary_qk(x, k, w, w, at, axes, norm="batch")
    with pytest.raises(ValueError, match="eps"):
        rot.norm_rotary_qk(x, k, w, w, at, axes, eps=-1.0)
    with pytest.raises(ValueError, match="k_weight"):
        rot.norm_rotary_qk(x, k, w, w[:7], at, axes)
    with pytest.raises(ValueError, match="q_bias"):
        rot.norm_rotary_qk(x, k, w, w, at, axes, q_bias=torch.ones(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="without a norm"):
        rot.norm_rotary_qk(x, k, w, w, at, axes, norm=None)
    qkv = torch.randn(2, 5, 64)
    with pytest.raises(ValueError, match="without a norm"):
        rot.rotary_attention_qkv(qkv, 4, 2, at, axes, q_weight=w)
    with pytest.raises(ValueError, match="divide"):
        rot.rotary_attention_qkv(qkv, 4, 3, at, axes)
    with pytest.raises(ValueError, match="window"):
        rot.rotary_attention_qkv(qkv, 4, 2, at, axes, window=-1)


@pytest.mark.parametrize("norm", [None, "layer", "rms"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,bands", [(6, (4,)), (8, (4, 4)), (10, (2, 6)), (16, (8, 4, 4))])
def test_cpu_formulation(norm, inter, D, bands):
    g = torch.Generator().manual_seed(3)
    axes = rot.RotaryAxes(bands, base=50.0, interleaved=inter)
    q, k = (torch.randn(2, 9, h, D, generator=g) for h in (4, 2))
    _check(q, k, axes, _grid(9, len(bands), "cpu"), norm, _params(D, "cpu", g) if norm else {})


def test_turns_are_relative_and_can_be_taken_back():
    torch.manual_seed(4)
    axes = rot.RotaryAxes((4, 8), base=30.0)
    q, k = torch.randn(6, 1, 14, dtype=torch.float64), torch.randn(6, 1, 14, dtype=torch.float64)
    at = torch.randint(0, 50, (6, 2))
    score = lambda s: torch.einsum("ihd,jhd->ij", *rot.rotary_qk(q, k, at + s, axes))  # noqa: E731
    assert torch.allclose(score(0), score(torch.tensor([17, -5])), atol=1e-10)
    assert torch.allclose(rot.rotary(rot.rotary(q, at, axes), at, axes, inverse=True), q, atol=1e-12)


def test_gradient_formulas_against_differences():
    torch.manual_seed(5)
    axes = rot.RotaryAxes((4, 2))
    x, w, b, do = torch.randn(5, 3, 8, dtype=torch.float64), torch.randn(8, dtype=torch.float64), torch.randn(8, dtype=torch.float64), None
    do = torch.randn_like(x)
    at = _grid(5, 2, "cpu")
    for norm in (None, "layer", "rms"):
        _, back = _oracle(x, w, b, at, axes, 1e-5, norm, do)
        f = lambda x, w, b: (_oracle(x, w, b, at, axes, 1e-5, norm)[0][0] * do).sum()  # noqa: E731,B023
        for i in range(3 if norm else 1):
            d = torch.randn_like((x, w, b)[i])
            up, down = ([t + s * 1e-6 * d if j == i else t for j, t in enumerate((x, w, b))] for s in (1, -1))
            assert abs((f(*up) - f(*down)).item() / 2e-6 - (back[i][0] * d).sum().item()) < 1e-6 * (1 + back[i][0].abs().sum().item())


# ---------------------------------------------------------------------------------------------------- the kernels

@pytest.fixture
def gen():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.available()
    before = _ext.launch_count()
    yield torch.Generator("cuda").manual_seed(11)
    torch.cuda.synchronize()
    assert _ext.launch_count() > before
    _ext.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "layer", "rms"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,N,H,Hk,D,bands", [
    (1, 1, 1, 1, 8, (8,)), (2, 128, 4, 4, 8, (4, 4)), (1, 37, 12, 3, 64, (32, 32)), (3, 50, 5, 1, 48, (24, 24)), (1, 1000, 8, 8, 128, (32, 48, 48)),
    (2, 19, 3, 3, 40, (10, 6, 4)), (1, 333, 7, 7, 72, (16, 40)), (1, 65, 2, 1, 136, (64, 8)), (1, 40, 6, 2, 256, (128, 64, 32, 32)), (1, 5000, 16, 4, 96, (16, 40, 32)),
    (1, 77, 9, 3, 24, (2,)), (37, 1, 16, 4, 128, (128,)),
    (1, 61, 3, 1, 40, (20, 20)), (2, 33, 5, 5, 72, (36, 12)), (1, 29, 6, 2, 256, (100, 4, 52)), (1, 51, 4, 2, 32, (4, 12)), (1, 90, 7, 1, 16, (6, 2))])
def test_widths_heads_and_lengths(gen, B, N, H, Hk, D, bands, dtype, inter, norm):
    axes = rot.RotaryAxes(bands, interleaved=inter)
    q, k = ((torch.randn(B, N, h, D, device="cuda", generator=gen) + 0.5).to(dtype) for h in (H, Hk))
    _check(q, k, axes, _grid(N, len(bands), "cuda"), norm, _params(D, "cuda", gen, bias=norm == "layer") if norm else {})


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32, torch.float64])
@pytest.mark.parametrize("per_sample", [False, True])
def test_positions(gen, kind, per_sample):
    """Far, negative and fractional positions; angles of position 10^7 in 32 bits would be off by a radian."""
    axes = rot.RotaryAxes((16, 16), base=(10000.0, 500.0))
    shape = (3, 21, 2) if per_sample else (21, 2)
    at = (torch.rand(shape, device="cuda", generator=gen, dtype=torch.float64) - 0.3) * 1e7
    q, k = (torch.randn(3, 21, h, 40, device="cuda", generator=gen) for h in (2, 1))
    _check(q, k, axes, at.to(kind), None, {})
    wide = torch.zeros(*shape[:-1], 4, device="cuda", dtype=kind)
    wide[..., ::2] = at.to(kind)
    assert torch.equal(rot.rotary(q, wide[..., ::2], axes), rot.rotary(q, at.to(kind), axes))


@pytest.mark.gpu
@pytest.mark.parametrize("inverse", [False, True])
def test_angles_next_to_quarters_of_a_turn(gen, inverse):
    """Sines and cosines that are small have as many right bits as others in bf16: half a step of the value, and what fp32 makes of a polynomial of five terms and
    its argument (4e-7 and eight roundings: 2^-19.8); angles are off by three roundings of 64 bits."""
    whole = [11, 22, 33, 355, 710, 1065, 103993, 104348, 208341, 312689, 833719]       # (next to multiples of pi)
    at = torch.tensor([0.0, 1e-7, 3e-6, -2e-5, 1e-4, -1e-3, 0.01, 0.3] + [float(s * n) for n in whole for s in (1, -1)] + [n / 2 + 1e-9 for n in whole],
                      dtype=torch.float64, device="cuda")
    axes = rot.RotaryAxes((2,), base=7.0)
    x = torch.zeros(2, at.numel(), 1, 8, device="cuda", dtype=torch.bfloat16)
    x[0, ..., 0] = 1.0
    x[1, ..., 1] = 1.0
    y = rot.rotary(x, at[:, None], axes, inverse=inverse)[:, :, 0, :2].double()
    turn = -at if inverse else at
    want = torch.stack([torch.stack([turn.cos(), turn.sin()], -1), torch.stack([-turn.sin(), turn.cos()], -1)])
    assert want.abs().min() == 0.0 and (want.abs() < 1e-4).sum() > 20
    assert ((y - want).abs() <= (2.0 ** -8 + 2.0 ** -19.8) * want.abs() + 3 * 2.0 ** -53 * at.abs()[:, None]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "layer", "rms"])
def test_strides_and_packed_tokens(gen, norm):
    """Views of a fused projection, heads in front, expanded and unaligned tensors, packed tokens."""
    axes = rot.RotaryAxes((16, 8))
    p = lambda: _params(32, "cuda", gen) if norm else {}  # noqa: E731
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731
    x = r(2, 30, 10, 32)
    at = _grid(30, 2, "cuda")
    _check(x[:, :, :6].detach(), x[:, :, 6:8].detach(), axes, at, norm, p())
    _check(r(2, 6, 30, 32).transpose(1, 2), r(30, 2, 2, 32).transpose(0, 1), axes, at, norm, p())
    _check(r(1, 30, 4, 32).expand(2, 30, 4, 32).detach(), r(2, 30, 1, 32).expand(2, 30, 3, 32).detach(), axes, at, norm, p())
    odd = r(2 * 30 * 4 * 32 + 1)[1:].view(2, 30, 4, 32)
    _check(odd.detach(), r(2, 30, 4, 33)[..., :32].detach(), axes, at, norm, p())
    _check(r(30, 4, 32), r(30, 2, 32), axes, at, norm, p())


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_norms_alone_and_parameters(gen, norm):
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).bfloat16()  # noqa: E731
    axes, at = rot.RotaryAxes((32,)), _grid(70, 1, "cuda")
    _check(r(2, 70, 4, 64), r(2, 70, 4, 64), None, None, norm, _params(64, "cuda", gen))
    _check(r(2, 70, 4, 64), r(2, 70, 2, 64), axes, at, norm, {})
    _check(r(2, 70, 4, 64), r(2, 70, 2, 64), axes, at, norm, _params(64, "cuda", gen, dtype=torch.bfloat16))
    only = _params(64, "cuda", gen)
    _check(r(2, 70, 4, 64), r(2, 70, 2, 64), axes, at, norm, dict(q_weight=only["q_weight"], k_bias=only["k_bias"]))
    # far from zero: the variance is that of deviations
    q, k = (r(1, 40, 3, 64).float() * 0.01 + 30.0 for _ in range(2))
    _check(q, k, axes, at[:40], norm, _params(64, "cuda", gen))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("N,H,Hk,D", [(37, 3, 1, 32), (1, 5, 5, 64), (131, 4, 3, 128), (9, 7, 2, 256)])
def test_no_eps(gen, N, H, Hk, D, norm):
    """Lanes that go along with zeros (behind the last token, head or sequence) have no standard deviation, and add nothing to the parameters' gradients."""
    axes, at = rot.RotaryAxes((16, 16)), _grid(N, 2, "cuda")
    q, k = (torch.randn(1, N, h, D, device="cuda", generator=gen).bfloat16() for h in (H, Hk))
    _check(q, k, axes, at, norm, _params(D, "cuda", gen), eps=0.0)
    if D > 128:
        return
    w = [torch.randn(D, device="cuda", generator=gen).requires_grad_() for _ in range(2)]
    qkv = torch.randn(N + 5, (H + 2 * Hk * (H % Hk == 0) + 2 * (H % Hk != 0)) * D, device="cuda", generator=gen).bfloat16()
    offsets, heads = torch.tensor([0, (N + 1) // 2, N], device="cuda", dtype=torch.int32), Hk if H % Hk == 0 else 1
    run = lambda x, at: rot.rotary_attention_qkv(x, H, heads, at, axes, *w, eps=0.0, norm=norm, offsets=offsets)  # noqa: E731
    o = run(qkv, _grid(N + 5, 2, "cuda"))
    got = torch.autograd.grad(o, w, torch.ones_like(o))
    o = run(qkv[:N], at)
    want = torch.autograd.grad(o, w, torch.ones_like(o))
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_partial_gradients(gen):
    """One result used, frozen inputs or parameters, none of them."""
    axes, at = rot.RotaryAxes((16, 16)), _grid(50, 2, "cuda")
    q, k = (torch.randn(1, 50, h, 32, device="cuda", generator=gen).bfloat16().requires_grad_() for h in (4, 2))
    p = {n: v.requires_grad_() for n, v in _params(32, "cuda", gen).items()}
    call = lambda q, k, **p: rot.norm_rotary_qk(q, k, p["q_weight"], p["k_weight"], at, axes, p["q_bias"], p["k_bias"])  # noqa: E731
    yq, yk = call(q, k, **p)
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    whole = torch.autograd.grad((yq, yk), [q, k, *p.values()], (dq, dk), retain_graph=True)
    alone = torch.autograd.grad(yk, [q, k, *p.values()], dk, retain_graph=True, allow_unused=True)
    for n, a, b in zip(["q", "k", *p], whole, alone):
        assert (b is None or not b.any()) if n[0] == "q" else torch.equal(a, b), n
    assert torch.equal(torch.autograd.grad((yq, yk), q, (dq, dk))[0], whole[0])
    frozen = call(q, k, **{n: v.detach() for n, v in p.items()})
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(frozen, (q, k), (dq, dk)), whole))
    params = call(q.detach(), k.detach(), **p)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(params, list(p.values()), (dq, dk)), whole[2:]))
    with torch.no_grad():
        assert torch.equal(call(q, k, **p)[0], yq) and not call(q, k, **p)[0].requires_grad


@pytest.mark.gpu
def test_no_tokens_and_infinities(gen):
    axes = rot.RotaryAxes((8,))
    w = torch.ones(16, device="cuda", requires_grad=True)
    for shape in ((0, 5, 2, 16), (2, 0, 2, 16), (2, 5, 0, 16)):
        q = torch.randn(*shape, device="cuda").bfloat16().requires_grad_()
        at = torch.zeros(shape[1], 1, device="cuda")
        y, _ = rot.norm_rotary_qk(q, torch.randn(*shape[:2], 2, 16, device="cuda").bfloat16(), w, w, at, axes)
        dq, dw = torch.autograd.grad(y, (q, w), torch.ones_like(y))
        assert y.shape == dq.shape == shape and not dw.any()
    # what is not turned stays as it is beside infinities, a row's NaN in its row
    for inter in (False, True):
        x = torch.randn(1, 6, 2, 16, device="cuda", generator=gen).bfloat16()
        x[0, 2, 1, 9] = math.inf
        x[0, 4, 0, 3] = math.nan
        y = rot.rotary(x, torch.arange(6, device="cuda")[:, None], rot.RotaryAxes((8,), interleaved=inter))
        assert torch.equal(y[..., 8:], x[..., 8:]) and torch.isfinite(y[..., :8]).sum() == 6 * 2 * 8 - 2


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,bands", [(8, (4, 4)), (16, None), (24, (8, 8)), (72, (36, 12)), (128, (128,)), (256, (64, 64))])
def test_norms_of_nan_and_infinities(gen, D, bands, dtype, norm):
    """A head with NaN or an infinity has the results that the definition gives it, NaN in every channel but where an infinite root mean square leaves zeros, the
    gradients of weights and biases with it; the other heads keep theirs."""
    axes, at = (None, None) if bands is None else (rot.RotaryAxes(bands), _grid(40, len(bands), "cuda"))
    p = {n: v.requires_grad_() for n, v in _params(D, "cuda", gen).items()}
    q, k = (torch.randn(1, 40, h, D, device="cuda", generator=gen).to(dtype).requires_grad_() for h in (5, 2))
    do = [torch.randn(t.shape, device="cuda", generator=gen).to(dtype) for t in (q, k)]

    def call(q, k):
        out = rot.norm_rotary_qk(q, k, p["q_weight"], p["k_weight"], at, axes, p["q_bias"], p["k_bias"], norm=norm)
        return out, torch.autograd.grad(out, [q, k, *p.values()], do)

    clean, clean_grads = call(q, k)
    heads = torch.ones(1, 40, 5, dtype=torch.bool, device="cuda")
    for value, channel in ((math.nan, 0), (math.nan, D - 1), (math.inf, 1), (-math.inf, D - 1)):
        bad = q.detach().clone()
        bad[0, 17, 3, channel] = value
        out, grads = call(bad.requires_grad_(), k)
        (want, _), back = _oracle(bad, p["q_weight"], p["q_bias"], at, axes, 1e-5, norm, do[0])
        heads[0, 17, 3] = False
        for n, got, w, before in (("q", out[0].detach(), want, clean[0].detach()), ("dq", grads[0], back[0][0], clean_grads[0])):
            assert torch.equal(got.isnan(), w.isnan()), (n, value)
            assert torch.equal(got[heads], before[heads]), (n, value)
            finite = ~w[0, 17, 3].isnan()
            assert w[0, 17, 3][finite].isfinite().all() and (norm == "rms" and n == "q" and abs(value) == math.inf or not finite.any())
            # (zeros, biases added and turned: off by A and F of two of these)
            _close(got[0, 17, 3][finite], w[0, 17, 3][finite], 2 * (A + F) * p["q_bias"].detach().abs().max(), n)
        # (of the weights; no bias has to do with what is normed)
        assert torch.equal(grads[2].isnan(), back[1][0].isnan()) and grads[2].isnan().any(), value
        assert torch.equal(grads[4], clean_grads[4])
        for i in (1, 3, 5):
            assert torch.equal(grads[i], clean_grads[i]), i


@pytest.mark.gpu
def test_rotation_can_be_differentiated_again(gen):
    axes, at = rot.RotaryAxes((8, 8)), _grid(9, 2, "cuda")
    x = torch.randn(1, 9, 2, 16, device="cuda", generator=gen).requires_grad_()
    y, _ = rot.rotary_qk(x, x[:, :, :1], at, axes)
    g, = torch.autograd.grad(y, x, y.detach(), create_graph=True)
    _, back = _oracle(x, None, None, at, axes, 0.0, None, y.detach())
    _close(g.detach(), *back[0], "dx")
    v = torch.randn_like(x)
    leaf = torch.randn_like(y).requires_grad_()
    g, = torch.autograd.grad(rot.rotary(x, at, axes), x, leaf, create_graph=True)
    gg, = torch.autograd.grad(g, leaf, v)
    assert torch.equal(gg, rot.rotary(v, at, axes))
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, _ = rot.norm_rotary_qk(x, x, w, w, at, axes)
    g, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


@pytest.mark.gpu
def test_transforms_see_through(gen):
    """`torch.func`, forward mode and tracing get torch's operations; batches of gradients are refused by name."""
    axes, at = rot.RotaryAxes((8, 8)), _grid(9, 2, "cuda")
    x = torch.randn(3, 9, 2, 16, device="cuda", generator=gen).bfloat16()
    y = rot.rotary(x, at, axes)
    many = torch.func.vmap(lambda t: rot.rotary(t, at, axes))(x)
    assert torch.allclose(many.float(), y.float(), atol=0.02)
    t = torch.randn_like(x)
    out, tangent = torch.func.jvp(lambda t: rot.rotary(t, at, axes), (x,), (t,))
    assert torch.allclose(tangent.float(), rot.rotary(t, at, axes).float(), atol=0.05)
    leaf = x.clone().requires_grad_()
    y = rot.rotary(leaf, at, axes)
    with pytest.raises(RuntimeError, match="batches of gradients"):
        torch.autograd.grad(y, leaf, torch.stack([y.detach()] * 2), is_grads_batched=True)
    compiled = torch.compile(lambda t: rot.rotary(t, at, axes), backend="eager")
    assert torch.allclose(compiled(x).float(), y.float(), atol=0.02)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "layer"])
def test_repeats_itself_and_replays(gen, norm):
    """The same bits every time, on another stream, and from a captured graph whose replays read the day's tensors and positions."""
    axes = rot.RotaryAxes((24, 24))
    q, k = (torch.randn(1, 3000, h, 48, device="cuda", generator=gen).bfloat16() for h in (8, 8))
    p = {n: v.requires_grad_() for n, v in _params(48, "cuda", gen).items()} if norm else {}
    at = _grid(3000, 2, "cuda")
    do = torch.randn(1, 3000, 8, 48, device="cuda", generator=gen).bfloat16()

    def call():
        a, b = (t.detach().requires_grad_() for t in (q, k))
        if norm:
            out = rot.norm_rotary_qk(a, b, p["q_weight"], p["k_weight"], at, axes, p["q_bias"], p["k_bias"])
        else:
            out = rot.rotary_qk(a, b, at, axes)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [a, b, *p.values()], (do, do)))

    first = call()
    assert all(torch.equal(a, b) for a, b in zip(first, call()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    with torch.no_grad():
        q.copy_(torch.randn_like(q))
        at.add_(5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, call()))


@pytest.mark.gpu
def test_many_tokens_of_one_head(gen):
    """Offsets past 32 bits: the last tokens of a strided tensor of more than 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.empty(2, 140000, 1, 8192, dtype=torch.bfloat16, device="cuda")
    q, k = x[..., :8], x[..., 4096:4104]
    q.normal_(generator=gen)
    k.normal_(generator=gen)
    axes = rot.RotaryAxes((8,))
    at = torch.arange(140000, device="cuda")[:, None]
    yq, yk = rot.rotary_qk(q, k, at, axes)
    for n, t, y in (("q", q, yq), ("k", k, yk)):
        (want, off), _ = _oracle(t[:, -100:], None, None, at[-100:], axes, 0.0, None)
        _close(y[:, -100:], want, off, n)


@pytest.mark.gpu
def test_refusals_on_the_device(gen):
    x, axes, at = torch.randn(1, 5, 2, 16, device="cuda").bfloat16(), rot.RotaryAxes((8, 8)), torch.zeros(5, 2, device="cuda")
    with pytest.raises(ValueError, match="positions"):
        rot.rotary(x, at.cpu(), axes)
    ext = _ext.require()
    none = [None] * 4
    with pytest.raises(RuntimeError, match="channels"):
        ext.rotary(x[..., :4], None, *none, at, axes.native(), 0, 0.0, False)
    with pytest.raises(RuntimeError, match="positions"):
        ext.rotary(x, None, *none, at[:4], axes.native(), 0, 0.0, False)
    with pytest.raises(RuntimeError, match="same tokens"):
        ext.rotary(x, x[:, :4], *none, at, axes.native(), 0, 0.0, False)
    with pytest.raises(RuntimeError, match="bf16 or fp32"):
        ext.rotary(x.half(), None, *none, at, axes.native(), 0, 0.0, False)
    with pytest.raises(RuntimeError, match="turned"):
        ext.rotary(x, None, *none, at, ext.RotaryPlan([8, 16], [0.0] * 12, False), 0, 0.0, False)
    # widths that the kernels do not have, and other types, through torch
    for t in (torch.randn(1, 5, 2, 10, device="cuda"), torch.randn(1, 5, 2, 16, device="cuda").half(), torch.randn(1, 5, 2, 16, device="cuda").double()):
        (want, off), _ = _oracle(t, None, None, at + 1, rot.RotaryAxes((4, 6)), 0.0, None)
        _close(rot.rotary(t, at + 1, rot.RotaryAxes((4, 6))), want, off, "other")
    rot.rotary(x, at, axes)
