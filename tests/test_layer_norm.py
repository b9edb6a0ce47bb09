"""Layer norm and layer norm behind a residual sum (`makani_b200/ops/norm.py`) against their definition in 64 bits.

Tolerances: outputs are rounded once, by at most half a step of their type.  Before that, sums of C values in fp32 lose at most some
SUM = 64 steps of 2^-24 of the sum of magnitudes (a thread adds up to 32 values, then five shuffles and eight warps), so that
xh = (x - mean) rstd is known to E = SUM 2^-24 (|xh| + mean|x| rstd), and everything below follows from E."""

import pytest
import torch

from makani_b200.ops import _ext
from makani_b200.ops import norm as norm_ops

U = 2.0 ** -24
SUM = 64


def _half_step(t):
    return torch.finfo(t).eps / 2


def _oracle(x, w, b, eps, dy=None):
    """In 64 bits on the device of x: y, dx, dw, db and how far each may be off before its rounding."""
    x, dy = x.double(), None if dy is None else dy.double()
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + b
    e = SUM * U * (xh.abs() + x.abs().mean(-1, keepdim=True) * rstd)
    out = dict(y=(y, e * w.abs() + 4 * U * (y.abs() + b.abs())))
    if dy is not None:
        g = dy * w
        m0, m1 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        dx = rstd * (g - m0 - xh * m1)
        gm, gx = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
        # rstd itself is known to SUM steps and what the mean's error moves it by, which e holds for |xh| = 1
        rel = SUM * U * (2 + x.abs().mean(-1, keepdim=True) * rstd)
        off = rstd * (SUM * U * (g.abs() + gm + xh.abs() * gx) + e * gx + xh.abs() * (g.abs() * e).mean(-1, keepdim=True) + rel * (g.abs() + gm + xh.abs() * gx))
        rows = x.numel() // C
        chain = rows / (148 * 8) + 400           # adds one after the other: a warp's rows, eight warps, the blocks
        red = tuple(range(x.dim() - 1))
        out["dx"] = (dx, off)
        out["dw"] = ((dy * xh).sum(red), (dy.abs() * e).sum(red) + chain * U * (dy * xh).abs().sum(red))
        out["db"] = (dy.sum(red), chain * U * dy.abs().sum(red))
    return out


def _close(got, want, what):
    val, off = want
    assert got.shape == val.shape, what
    diff = (got.double() - val).abs()
    bound = off * (1 + _half_step(got.dtype)) + _half_step(got.dtype) * val.abs() + 1e-37
    bad = ~(diff <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((diff / bound)[bad].max()):.2f} of the bound"


def _tokens(g, *shape, dtype=torch.bfloat16, mean=1.0, device="cuda"):
    C = shape[-1]
    loc = mean * torch.randn(C, device=device, generator=g)
    return (torch.randn(*shape, device=device, generator=g) * (0.5 + torch.rand(C, device=device, generator=g)) + loc).to(dtype)


def _check(x, w, b, dy, out_dtype, eps=1e-5, residual=None, ds=None):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, residual) if t is not None]
    it = iter(leaves)
    xl = next(it)
    wl = None if w is None else next(it)
    bl = None if b is None else next(it)
    rl = None if residual is None else next(it)
    if residual is None:
        y = norm_ops.layer_norm(xl, wl, bl, eps, out_dtype)
        grads = torch.autograd.grad(y, leaves, dy)
        source = x
    else:
        s, y = norm_ops.add_layer_norm(xl, rl, wl, bl, eps, out_dtype)
        assert s.dtype == torch.promote_types(x.dtype, residual.dtype)
        assert torch.equal(s, x + residual)      # one rounding of an fp32 sum, as torch's
        grads = torch.autograd.grad((s, y), leaves, (ds, dy))
        source = s.detach()
    assert y.dtype == (out_dtype or source.dtype) and y.is_contiguous()
    want = _oracle(source, w, b, eps, dy)
    _close(y.detach(), want["y"], "y")
    dx, off = want["dx"]
    if ds is not None:
        dx = dx + ds.double()
        off = off + 2 * U * (dx.abs() + ds.double().abs())
    assert grads[0].dtype == x.dtype
    _close(grads[0], (dx, off), "dx")
    if rl is not None:
        assert grads[-1].dtype == residual.dtype
        _close(grads[-1], (dx, off), "dr")
    at = 1
    for name, p in (("dw", w), ("db", b)):
        if p is not None:
            assert grads[at].dtype == p.dtype
            _close(grads[at], want[name], name)
            at += 1


# ---------------------------------------------------------------------------------------------------- any machine

def test_refusals():
    x = torch.randn(4, 16)
    w, b = torch.ones(16), torch.zeros(16)
    with pytest.raises(ValueError, match="weight"):
        norm_ops.layer_norm(x, torch.ones(8), b)
    with pytest.raises(ValueError, match="bias"):
        norm_ops.layer_norm(x, w, torch.zeros(1, 16))
    with pytest.raises(ValueError, match="floating"):
        norm_ops.layer_norm(x.long(), w, b)
    with pytest.raises(ValueError, match="floating"):
        norm_ops.layer_norm(torch.randn(()), None, None)
    with pytest.raises(ValueError, match="output"):
        norm_ops.layer_norm(x, w, b, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="residual"):
        norm_ops.add_layer_norm(x, x[:2], w, b)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
def test_cpu_formulation(dtype):
    g = torch.Generator().manual_seed(3)
    x, r = _tokens(g, 3, 7, 20, dtype=dtype, device="cpu"), _tokens(g, 3, 7, 20, dtype=dtype, device="cpu")
    w, b = torch.randn(20, generator=g), torch.randn(20, generator=g)
    _close(norm_ops.layer_norm(x, w, b, 1e-6), _oracle(x, w, b, 1e-6)["y"], "y")
    s, y = norm_ops.add_layer_norm(x, r, w, b, 1e-6, out_dtype=torch.float32)
    assert torch.equal(s, x + r) and y.dtype == torch.float32
    _close(y, _oracle(s, w, b, 1e-6)["y"], "y")


def test_gradient_formula_against_differences():
    """The formulas that the oracle holds the kernels to are the derivatives of the definition."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 9, generator=g, dtype=torch.float64)
    w, b, dy, d = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((9,), (9,), (3, 9), (3, 9)))
    want = _oracle(x, w, b, 1e-5, dy)
    f = lambda x_, w_, b_: (_oracle(x_, w_, b_, 1e-5)["y"][0] * dy).sum()  # noqa: E731
    h = 1e-5
    for got, plus, minus in (((want["dx"][0] * d).sum(), f(x + h * d, w, b), f(x - h * d, w, b)),
                             ((want["dw"][0] * d[0]).sum(), f(x, w + h * d[0], b), f(x, w - h * d[0], b)),
                             ((want["db"][0] * d[0]).sum(), f(x, w, b + h * d[0]), f(x, w, b - h * d[0]))):
        assert abs(float(got - (plus - minus) / (2 * h))) < 1e-8 * (1 + abs(float(got)))


# ---------------------------------------------------------------------------------------------------- the kernels

@pytest.fixture
def gen():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.available()
    return torch.Generator("cuda").manual_seed(11)


SIZES = [(1, 8), (3, 1), (5, 7), (33, 48), (1000, 56), (129, 64), (257, 72), (31, 128), (70, 200), (1, 256), (300, 384), (7, 387), (41, 512), (1201, 520),
         (19, 768), (6, 1000), (23, 1024), (77, 1023), (9, 1032), (150, 2048), (5, 2050), (3, 8192), (2, 8191), (40000, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", SIZES)
@pytest.mark.parametrize("xt,yt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float32, torch.float32),
                                   (torch.bfloat16, torch.float32)])
def test_layer_norm(gen, rows, C, xt, yt):
    x, dy = _tokens(gen, rows, C, dtype=xt), torch.randn(rows, C, device="cuda", generator=gen).to(yt)
    w, b = 1 + 0.2 * torch.randn(C, device="cuda", generator=gen), 0.2 * torch.randn(C, device="cuda", generator=gen)
    _check(x, w, b, dy, yt)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", [(1, 8), (33, 48), (300, 384), (7, 387), (23, 1024), (9, 1032), (2, 8191)])
@pytest.mark.parametrize("xt,rt,yt", [(torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16, torch.bfloat16),
                                      (torch.float32, torch.float32, torch.float32), (torch.float32, torch.bfloat16, torch.float32)])
def test_add_layer_norm(gen, rows, C, xt, rt, yt):
    x, r = _tokens(gen, rows, C, dtype=xt), _tokens(gen, rows, C, dtype=rt)
    dy, ds = torch.randn(rows, C, device="cuda", generator=gen).to(yt), torch.randn(rows, C, device="cuda", generator=gen).to(xt)
    w, b = 1 + 0.2 * torch.randn(C, device="cuda", generator=gen), 0.2 * torch.randn(C, device="cuda", generator=gen)
    _check(x, w, b, dy, yt, residual=r, ds=ds)


@pytest.mark.gpu
def test_add_layer_norm_either_order_and_parts(gen):
    x, r = _tokens(gen, 50, 64, dtype=torch.bfloat16), _tokens(gen, 50, 64, dtype=torch.float32)
    w = torch.ones(64, device="cuda")
    a, b = norm_ops.add_layer_norm(x, r, w, None), norm_ops.add_layer_norm(r, x, w, None)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[0].dtype == a[1].dtype == torch.float32
    # the gradient of the sum alone, and of the norm alone
    xl, rl = x.clone().requires_grad_(), r.clone().requires_grad_()
    s, y = norm_ops.add_layer_norm(xl, rl, w, None)
    gx, gr = torch.autograd.grad(s.sum(), (xl, rl), retain_graph=True)
    assert gx.dtype == torch.bfloat16 and torch.equal(gx, torch.ones_like(gx)) and torch.equal(gr, torch.ones_like(gr))
    dy = torch.randn(50, 64, device="cuda", generator=gen)
    gx, gr = torch.autograd.grad(y, (xl, rl), dy)
    want = _oracle(s.detach(), w, None, 1e-5, dy)["dx"]
    _close(gx, want, "dx")
    _close(gr, want, "dr")


@pytest.mark.gpu
@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
def test_without_parameters(gen, w, b):
    x, dy = _tokens(gen, 37, 96), torch.randn(37, 96, device="cuda", generator=gen).bfloat16()
    p = torch.randn(96, device="cuda", generator=gen)
    _check(x, p if w else None, p.flip(0) if b else None, dy, None)


@pytest.mark.gpu
def test_parameters_in_bf16(gen):
    x, dy = _tokens(gen, 37, 96), torch.randn(37, 96, device="cuda", generator=gen).bfloat16()
    _check(x, (1 + torch.randn(96, device="cuda", generator=gen)).bfloat16(), torch.randn(96, device="cuda", generator=gen).bfloat16(), dy, None)


@pytest.mark.gpu
def test_strided_rows(gen):
    B, N, H, D = 2, 19, 5, 24
    w, b = torch.randn(D, device="cuda", generator=gen), torch.randn(D, device="cuda", generator=gen)
    dy = torch.randn(B, N, H, D, device="cuda", generator=gen).bfloat16()
    qkv = _tokens(gen, B, N, 3, H, D)
    _check(qkv[:, :, 1], w, b, dy, None)                                           # two levels
    _check(qkv[:, :, 2].transpose(1, 2), w, b, dy.transpose(1, 2), None)           # three: copied
    _check(qkv[:, :, 0, 1:2].expand(B, N, H, D), w, b, dy, None)                   # one row seen by several
    _check(_tokens(gen, B, N, H, 2 * D)[..., ::2], w, b, dy, None)                 # elements apart: copied
    _check(_tokens(gen, B * N * H * D + 1)[1:].view(B, N, H, D), w, b, dy, None)   # off a 16-byte boundary
    _check(_tokens(gen, B, N, H, D + 1)[..., :D], w, b, dy, None)                  # rows off a 16-byte boundary


@pytest.mark.gpu
def test_far_mean_and_constant_rows(gen):
    """|mean| = 300 spreads: a variance from E[x^2] - E[x]^2 would be lost; constant rows give the bias."""
    x = (300 + torch.randn(64, 384, device="cuda", generator=gen)).float()
    x[7] = 5.0
    w, b = torch.randn(384, device="cuda", generator=gen), torch.randn(384, device="cuda", generator=gen)
    dy = torch.randn(64, 384, device="cuda", generator=gen)
    y = norm_ops.layer_norm(x, w, b)
    assert torch.equal(y[7], b)
    keep = torch.arange(64, device="cuda") != 7
    _check(x[keep], w, b, dy[keep], torch.float32)


@pytest.mark.gpu
def test_infinities_stay_in_their_rows(gen):
    x = _tokens(gen, 70, 72)
    x[3, 5], x[11, 0] = float("nan"), float("inf")
    w, b = torch.ones(72, device="cuda"), torch.zeros(72, device="cuda")
    y = norm_ops.layer_norm(x, w, b)
    bad = torch.tensor([3, 11], device="cuda")
    assert y[bad].isnan().all()
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[bad] = False
    _close(y[keep], _oracle(x[keep], w, b, 1e-5)["y"], "y")


@pytest.mark.gpu
def test_no_rows(gen):
    x = torch.empty(0, 3, 40, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w, b = torch.ones(40, device="cuda", requires_grad=True), torch.zeros(40, device="cuda", requires_grad=True)
    y = norm_ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.gpu
def test_repeats_itself_and_replays(gen):
    """The same bits again, on another stream, and from a captured graph with new inputs."""
    x, dy = _tokens(gen, 5000, 384), torch.randn(5000, 384, device="cuda", generator=gen).bfloat16()
    w, b = torch.randn(384, device="cuda", generator=gen).requires_grad_(), torch.randn(384, device="cuda", generator=gen).requires_grad_()

    def both(xi):
        xl = xi.detach().requires_grad_()
        y = norm_ops.layer_norm(xl, w, b)
        return (y.detach(),) + torch.autograd.grad(y, (xl, w, b), dy)

    first = both(x)
    assert all(torch.equal(p, q) for p, q in zip(first, both(x)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(p, q) for p, q in zip(first, both(x)))
        xs = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = both(xs)
    torch.cuda.current_stream().wait_stream(side)
    for k in (1, 2):
        xs.copy_(x.roll(k, 0))
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, both(x.roll(k, 0))))
    del graph


@pytest.mark.gpu
def test_difference_quotient(gen):
    """The kernel's own outputs, a step to either side, against its gradient; what the step leaves out is taken from 64 bits."""
    x, dy, d = _tokens(gen, 40, 200, dtype=torch.float32), *(torch.randn(40, 200, device="cuda", generator=gen) for _ in range(2))
    w, b, h = torch.randn(200, device="cuda", generator=gen), torch.randn(200, device="cuda", generator=gen), 2.0 ** -6
    xl = x.clone().requires_grad_()
    dx = torch.autograd.grad(norm_ops.layer_norm(xl, w, b), xl, dy)[0]
    f = lambda fn, t: (fn(t).double() * dy.double()).sum()  # noqa: E731
    own = lambda t: norm_ops.layer_norm(t, w, b)  # noqa: E731
    ref = lambda t: _oracle(t, w, b, 1e-5)["y"][0]  # noqa: E731
    up, down = x + h * d, x - h * d
    quotient = (f(own, up) - f(own, down)) / (2 * h)
    left_out = (f(ref, up) - f(ref, down)) / (2 * h) - (_oracle(x, w, b, 1e-5, dy)["dx"][0] * d.double()).sum()
    off = sum((_oracle(t, w, b, 1e-5)["y"][1] * dy.double().abs()).sum() for t in (up, down)) / (2 * h)
    assert abs(float(quotient - left_out - (dx.double() * d.double()).sum())) <= float(off) + 1e-3


@pytest.mark.gpu
def test_kernels_are_counted(gen):
    x = _tokens(gen, 64, 64).requires_grad_()
    before = _ext.launch_count()
    norm_ops.layer_norm(x, torch.ones(64, device="cuda", requires_grad=True), None).sum().backward()
    assert _ext.launch_count() > before


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("xt,wt", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_second_derivatives(gen, residual, xt, wt):
    """Gradients that are differentiated once more, against 64 bits.  A first gradient in fp32 is known to E = SUM U of the magnitudes it is made of; a second one
    is made of products of some four such quantities, sums of them, and one sum more over the rows for the weight: 16 E = 6.1e-5 of its norm.  In bf16 the
    first gradient is rounded, as torch's is, and what comes back through that rounding too: three roundings of half a step."""
    C, rows = 40, 9
    x = _tokens(gen, rows, C, dtype=xt).requires_grad_()
    r = _tokens(gen, rows, C, dtype=xt).requires_grad_() if residual else None
    w = (1 + 0.2 * torch.randn(C, device="cuda", generator=gen)).to(wt).requires_grad_()
    b = torch.zeros(C, device="cuda", dtype=wt, requires_grad=True)
    dy = torch.randn(rows, C, device="cuda", generator=gen).to(xt).requires_grad_()
    ds = torch.randn(rows, C, device="cuda", generator=gen).to(xt)
    tx, tw, tb = (torch.randn(s, device="cuda", generator=gen) for s in ((rows, C), (C,), (C,)))

    def second(f, x, r, w, b, dy, ds):
        s, y = f(x, r, w, b)
        first = torch.autograd.grad((s, y) if residual else y, (x, w, b), (ds, dy) if residual else dy, create_graph=True)
        work = torch.promote_types(s.dtype, torch.float32)
        score = sum((g.to(work) * t.to(work)).sum() for g, t in zip(first, (tx, tw, tb)))
        leaves = [t for t in (x, r, w, dy) if t is not None]
        return torch.autograd.grad(score, leaves)

    def own(x, r, w, b):
        return norm_ops.add_layer_norm(x, r, w, b, 1e-5, xt) if residual else (x, norm_ops.layer_norm(x, w, b, 1e-5, xt))

    def definition(x, r, w, b):
        s = x + r if residual else x
        if residual and xt == torch.bfloat16:
            s = s + (s.detach().bfloat16().double() - s.detach())       # the sum is rounded; its gradient is not
        mean = s.mean(-1, keepdim=True)
        return s, (s - mean) / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + 1e-5) * w + b

    got = second(own, x, r, w, b, dy, ds)
    want = second(definition, *(None if t is None else t.detach().double().requires_grad_() for t in (x, r, w, b, dy)), ds.double())
    for g, t in zip(got, want):
        off = 16 * SUM * U + (3 * _half_step(torch.bfloat16) if torch.bfloat16 in (xt, wt) else 0)
        assert (g.double() - t).norm() <= off * t.norm(), (g.shape, float((g.double() - t).norm() / t.norm()))


@pytest.mark.gpu
def test_transforms_see_through_the_norms(gen):
    """vmap, forward mode, tracing, compilation and fake tensors go by torch's operations, as with `nn.LayerNorm`."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, d, r = (torch.randn(4, 6, 24, device="cuda", generator=gen) for _ in range(3))
    w, b = torch.randn(24, device="cuda", generator=gen), torch.randn(24, device="cuda", generator=gen)
    own = lambda t: norm_ops.layer_norm(t, w, b)  # noqa: E731
    added = lambda t: norm_ops.add_layer_norm(t, r[0] if t.dim() == 2 else r, w, b)[1]  # noqa: E731
    plain = lambda t: torch.nn.functional.layer_norm(t, (24,), w, b)  # noqa: E731
    near = lambda p, q: torch.allclose(p, q, rtol=1e-5, atol=1e-5)  # noqa: E731
    assert near(torch.func.vmap(own)(x), plain(x))
    assert near(torch.func.vmap(added)(x), plain(x + r[0]))
    assert near(torch.func.jacrev(lambda t: own(t).sum(0))(x[0, 0][None]), torch.func.jacrev(lambda t: plain(t).sum(0))(x[0, 0][None]))
    for f, g in ((own, plain), (added, lambda t: plain(t + r))):
        y, dy = torch.func.jvp(f, (x,), (d,))
        y0, dy0 = torch.func.jvp(g, (x,), (d,))
        assert near(y, y0) and near(dy, dy0)
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x, d)
            assert near(torch.autograd.forward_ad.unpack_dual(f(dual)).tangent, dy0)
        traced = torch.jit.trace(f, (x,))
        assert near(traced(d), g(d))
        assert near(torch.compile(f, backend="eager", fullgraph=True)(d), g(d))
        assert near(make_fx(f)(x)(d), g(d))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        fake = mode.from_tensor(x)
        y = norm_ops.layer_norm(fake, None, None)
    assert y.shape == x.shape


# Groups that go over three rows or sets of rows and more, the last turn ragged
@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", [(10007, 384), (5003, 1024), (2501, 387), (40001, 48), (20011, 120), (1501, 2056), (701, 2051), (1203, 8192)])
@pytest.mark.parametrize("xt,rt,yt", [(torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.bfloat16, torch.float32),
                                      (torch.float32, torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16, torch.float32),
                                      (torch.float32, torch.float32, torch.bfloat16), (torch.float32, torch.float32, torch.float32)])
def test_add_layer_norm_of_several_turns(gen, rows, C, xt, rt, yt):
    x, r = _tokens(gen, rows, C, dtype=xt), _tokens(gen, rows, C, dtype=rt)
    dy, ds = torch.randn(rows, C, device="cuda", generator=gen).to(yt), torch.randn(rows, C, device="cuda", generator=gen).to(xt)
    w, b = 1 + 0.2 * torch.randn(C, device="cuda", generator=gen), 0.2 * torch.randn(C, device="cuda", generator=gen)
    _check(x, w, b, dy, yt, residual=r, ds=ds)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", [(15001, 384), (7001, 1024), (3001, 387), (60001, 40), (2003, 2056)])
@pytest.mark.parametrize("xt,yt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float32, torch.float32),
                                   (torch.bfloat16, torch.float32)])
def test_layer_norm_of_several_turns(gen, rows, C, xt, yt):
    x, dy = _tokens(gen, rows, C, dtype=xt), torch.randn(rows, C, device="cuda", generator=gen).to(yt)
    w, b = 1 + 0.2 * torch.randn(C, device="cuda", generator=gen), 0.2 * torch.randn(C, device="cuda", generator=gen)
    _check(x, w, b, dy, yt)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", [(1, 8), (64, 48), (700, 128), (333, 387), (5001, 768), (90, 1024), (41, 1023), (70, 1032), (9, 2051), (12, 4096)])
@pytest.mark.parametrize("wt,bt", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float64),
                                   (torch.bfloat16, None), (None, torch.bfloat16)])
def test_types_of_parameters(gen, rows, C, wt, bt):
    """Weights and biases in types of their own, each with its gradient rounded once to its type, by one block and by several."""
    x, dy = _tokens(gen, rows, C), torch.randn(rows, C, device="cuda", generator=gen).bfloat16()
    w = None if wt is None else (1 + 0.2 * torch.randn(C, device="cuda", generator=gen)).to(wt)
    b = None if bt is None else (0.2 * torch.randn(C, device="cuda", generator=gen)).to(bt)
    _check(x, w, b, dy, None)
    _check(x, w, b, dy, torch.bfloat16, residual=_tokens(gen, rows, C), ds=dy.flip(0))
    if wt is not None and C > 8:      # off a 16-byte boundary
        _check(x, torch.cat([w[:1], w])[1:], b, dy, None)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["norm", "sum and norm", "sum", "behind a sum"])
def test_compiled_backward_pass(gen, which):
    """The backward pass that is compiled calls the kernels: the same bits."""
    from torch._dynamo import compiled_autograd
    x, r = (torch.randn(9, 40, device="cuda", generator=gen).requires_grad_() for _ in range(2))
    w = torch.randn(40, device="cuda", generator=gen).bfloat16().requires_grad_()

    def grads():
        s, y = norm_ops.add_layer_norm(x, r, w, None)
        if which == "norm":
            y = norm_ops.layer_norm(x, w, None)
        out = {"norm": y, "sum and norm": s * s + y * y, "sum": s * s, "behind a sum": y * y}[which]
        return torch.autograd.grad(out.sum(), (x, r, w), allow_unused=True)

    want = grads()
    with compiled_autograd._enable(torch.compile(backend="eager")):
        got = grads()
    for p, q in zip(got, want):
        assert (p is None and q is None) or torch.equal(p, q)


@pytest.mark.gpu
def test_a_second_backward_pass(gen):
    x = torch.randn(9, 40, device="cuda", generator=gen).requires_grad_()
    s, y = norm_ops.add_layer_norm(x, x, None, None)
    first = torch.autograd.grad(y.sum() + s.sum(), x, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y.sum() + s.sum(), x)[0])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y.sum(), x)
    s, y = norm_ops.add_layer_norm(x, x, None, None)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
def test_transforms_of_the_backward_pass(gen, residual):
    """Batches of output gradients and traces of a backward pass, through a graph that the kernels made."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, r, dy = (torch.randn(7, 24, device="cuda", generator=gen) for _ in range(3))
    w = torch.randn(24, device="cuda", generator=gen).requires_grad_()
    leaves = [t.requires_grad_() for t in ((x, r) if residual else (x,))] + [w]
    y = norm_ops.add_layer_norm(x, r, w, None)[1] if residual else norm_ops.layer_norm(x, w, None)
    batch = torch.randn(5, 7, 24, device="cuda", generator=gen)
    got = torch.autograd.grad(y, leaves, batch, is_grads_batched=True, retain_graph=True)
    for i in range(5):
        for g, t in zip(got, torch.autograd.grad(y, leaves, batch[i], retain_graph=True)):
            assert torch.allclose(g[i], t, rtol=1e-5, atol=1e-5)
    back = lambda d: torch.autograd.grad(y, leaves, d, retain_graph=True)  # noqa: E731
    traced = make_fx(back)(dy)
    for g, t in zip(traced(batch[0]), back(batch[0])):
        assert torch.allclose(g, t, rtol=1e-5, atol=1e-5)
