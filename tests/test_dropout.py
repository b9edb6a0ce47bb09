"""Dropout from a counter (`makani_b200/ops/dropout.py`): the generator against the published algorithm in whole numbers of any size, the mask bit for bit,
values to half a step of their type (and the fp32 steps of factor, product and sum before it)."""

import math

import pytest
import torch

from makani_b200.ops import _ext
from makani_b200.ops import dropout as drop


def _philox(counter, key):
    """Philox4x32 with ten rounds in Python's whole numbers."""
    c, k, m = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def _words(key, number, elements):
    split = lambda v: [v & 0xFFFFFFFF, (v >> 32) & 0xFFFFFFFF]  # noqa: E731
    return [_philox(split(number) + split(i >> 2), split(key))[i & 3] for i in elements]


def _keep(seed, shape, p, device):
    n = math.prod(shape)
    return (drop.random_words(seed.cpu(), n) >= round(p * 2 ** 32)).view(shape).to(device)


def _close(got, want, magnitude, what):
    bound = 2.0 ** -21 * magnitude + torch.finfo(got.dtype).eps / 2 * want.abs() + 1e-40
    assert ((got.double() - want).abs() <= bound * (1 + 2.0 ** -8)).all(), what


def _check(x, p, seed, residual=None, dy=None):
    leaves = [t.detach().requires_grad_() for t in (x, residual) if t is not None]
    y = drop.dropout(leaves[0], p, seed=seed) if residual is None else drop.dropout_add(*leaves, p, seed=seed)
    dy = torch.randn_like(y) if dy is None else dy
    grads = torch.autograd.grad(y, leaves, dy)
    keep = _keep(seed, x.shape, p, x.device)
    f = 1 / (1 - p) if p < 1 else 0.0
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    want = torch.where(keep, x.double() * f, zero)
    r = zero if residual is None else residual.double()
    assert y.dtype == (x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)) and y.shape == x.shape
    _close(y.detach(), want + r, want.abs() + r.abs(), "y")
    if residual is None:
        assert not y.detach()[~keep].any()
    want = torch.where(keep, dy.double() * f, zero)
    assert grads[0].dtype == x.dtype and not grads[0][~keep].any()
    _close(grads[0], want, want.abs(), "dx")
    if residual is not None:
        assert torch.equal(grads[1], dy.to(residual.dtype))
    return y.detach(), grads


# ---------------------------------------------------------------------------------------------------- any machine

def test_generator():
    # known answers of the algorithm as published (counter, key: all zeros, all ones)
    assert _philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    for key, number in ((0, 0), (1, 2), (-1, -7), (2 ** 62 + 5, 2 ** 40 + 1)):
        got = drop.random_words(torch.tensor([key, number]), 103).tolist()
        assert got == _words(key, number, range(103))


def test_refusals():
    x, seed = torch.randn(5), torch.tensor([1, 2])
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="probability"):
            drop.dropout(x, p)
    with pytest.raises(ValueError, match="floating"):
        drop.dropout(x.long())
    for bad in (seed.int(), seed[:1], seed[None]):
        with pytest.raises(ValueError, match="seed"):
            drop.dropout(x, 0.5, seed=bad)
    for bad in (torch.randn(4), torch.randn(5).long(), torch.randn(1, 5)):
        with pytest.raises(ValueError, match="residual"):
            drop.dropout_add(x, bad, 0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_cpu_formulation(dtype):
    torch.manual_seed(1)
    x, r, seed = torch.randn(3, 7, dtype=dtype), torch.randn(3, 7), torch.tensor([5, 9])
    for p in (0.1, 0.5, 1.0):
        _check(x, p, seed)
        _check(x, p, seed, r)
    assert drop.dropout(x, 0.0) is x and drop.dropout(x, 0.3, training=False) is x
    assert torch.equal(drop.dropout_add(x, r, 0.3, training=False), x + r)
    torch.manual_seed(2)
    y = drop.dropout(torch.ones(4000), 0.25)
    assert set(y.unique().tolist()) == {0.0, torch.tensor(1.0).div(0.75).item()} and abs((y == 0).double().mean() - 0.25) < 0.05


# ---------------------------------------------------------------------------------------------------- the kernel

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


PAIRS = [(torch.bfloat16, None), (torch.float32, None), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
         (torch.float32, torch.float32)]


@pytest.mark.gpu
@pytest.mark.parametrize("x_type,r_type", PAIRS)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (2047,), (2049,), (3, 5, 17), (129, 768), (100003,)])
def test_sizes_and_types(gen, shape, x_type, r_type):
    seed = torch.tensor([2 ** 50 + 3, 17], device="cuda")
    x = torch.randn(shape, device="cuda", generator=gen).to(x_type)
    r = None if r_type is None else torch.randn(shape, device="cuda", generator=gen).to(r_type)
    for p in (0.1, 0.9):
        _check(x, p, seed, r)


@pytest.mark.gpu
def test_seeds_and_probabilities(gen):
    x = torch.ones(4 * 999, device="cuda")
    for key, number in ((0, 0), (-1, -1), (2 ** 63 - 1, 2 ** 40)):
        _check(x, 0.5, torch.tensor([key, number], device="cuda"))
    seed = torch.tensor([3, 4], device="cuda")
    for p in (2.0 ** -31, 1e-6, 0.3, 1 - 2.0 ** -20, 1 - 1e-12, 1.0):
        _check(x, p, seed)
    assert drop.dropout(x, 2.0 ** -40, seed=seed) is x
    few = drop.dropout(torch.ones(1 << 22, device="cuda"), 0.01, seed=seed)
    # (a binomial: five standard deviations)
    assert abs((few == 0).double().mean().item() - 0.01) < 5 * math.sqrt(0.01 * 0.99 / (1 << 22))


@pytest.mark.gpu
def test_strides_alignment_and_infinities(gen):
    seed = torch.tensor([3, 4], device="cuda")
    x = torch.randn(40, 50, device="cuda", generator=gen).bfloat16()
    a = drop.dropout(x.t(), 0.4, seed=seed)
    assert torch.equal(a, drop.dropout(x.t().contiguous(), 0.4, seed=seed))
    flat = torch.randn(1001, device="cuda", generator=gen).bfloat16()
    _check(flat[1:], 0.4, seed)
    _check(flat[:1000], 0.4, seed, torch.randn(1003, device="cuda")[3:])
    _check(x[:, ::2], 0.4, seed, torch.randn(1, 25, device="cuda").expand(40, 25))
    keep = _keep(seed, (64,), 0.4, "cuda")
    bad = torch.full((64,), math.nan, device="cuda").masked_fill(keep, 1.0)
    y, _ = _check(bad.nan_to_num(0.0), 0.4, seed)
    assert torch.equal(drop.dropout(bad, 0.4, seed=seed), y)
    assert drop.dropout(torch.empty(0, 3, device="cuda"), 0.4).shape == (0, 3)
    e = torch.empty(0, 3, device="cuda", requires_grad=True)
    drop.dropout_add(e, e, 0.4).sum().backward()


@pytest.mark.gpu
def test_torchs_generator(gen):
    """Seeds of torch's generator: repeatable, new from call to call, apart from those of torch's own random numbers, and the backward pass has the forward's."""
    x = torch.ones(100000, device="cuda", requires_grad=True)

    def calls():
        torch.manual_seed(7)
        a = drop.dropout(x, 0.5)
        u = torch.rand(100000, device="cuda")
        b = drop.dropout(x, 0.5)
        ga, = torch.autograd.grad(a, x, torch.ones_like(a), retain_graph=True)
        gb, = torch.autograd.grad(b, x, torch.ones_like(b))
        return a.detach(), u, b.detach(), ga, gb

    first, again = calls(), calls()
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    a, u, b, ga, gb = first
    assert torch.equal(a, ga) and torch.equal(b, gb)
    for p, q in ((a > 0, b > 0), (a > 0, u > 0.5), (b > 0, u > 0.5)):      # (independent: half of them agree)
        assert abs((p == q).double().mean().item() - 0.5) < 0.01
    # a checkpointed pass draws the same mask again
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(9)
    y = checkpoint(lambda t: drop.dropout(t, 0.5) * t, x, use_reentrant=False)
    g, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, 2 * y.detach())


@pytest.mark.gpu
def test_captured_graphs_draw_new_masks(gen):
    x = torch.ones(50000, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        y = drop.dropout(x, 0.5)
        torch.autograd.grad(y, x, torch.ones_like(y))
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            y = drop.dropout(x, 0.5)
            z = drop.dropout(x, 0.5)
            g, h = (torch.autograd.grad(t, x, torch.ones_like(t))[0] for t in (y, z))
    torch.cuda.synchronize()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), g) and torch.equal(z.detach(), h)
        seen += [g.clone() > 0, h.clone() > 0]
    for i, a in enumerate(seen):
        assert abs(a.double().mean().item() - 0.5) < 0.02
        for b in seen[:i]:
            assert abs((a == b).double().mean().item() - 0.5) < 0.02


@pytest.mark.gpu
def test_gradients_can_be_differentiated_again(gen):
    seed = torch.tensor([3, 4], device="cuda")
    for x_type, r_type in PAIRS:
        x = torch.randn(300, device="cuda", generator=gen).to(x_type).requires_grad_()
        r = None if r_type is None else torch.randn(300, device="cuda", generator=gen).to(r_type).requires_grad_()
        y = drop.dropout(x, 0.5, seed=seed) if r is None else drop.dropout_add(x, r, 0.5, seed=seed)
        dy = torch.randn_like(y).requires_grad_()
        g = torch.autograd.grad(y, x if r is None else (x, r), dy, create_graph=True)
        want, = torch.autograd.grad(g[0], dy, torch.ones_like(g[0]))
        keep = _keep(seed, (300,), 0.5, "cuda")
        assert torch.equal(want.float(), 2.0 * keep.float())


@pytest.mark.gpu
def test_partial_gradients_and_transforms(gen):
    seed = torch.tensor([3, 4], device="cuda")
    x, r = torch.randn(500, device="cuda", generator=gen).bfloat16(), torch.randn(500, device="cuda", generator=gen)
    y = drop.dropout_add(x, r.requires_grad_(), 0.5, seed=seed)
    dy = torch.randn_like(y)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)
    half = r.detach().bfloat16().requires_grad_()
    assert torch.equal(torch.autograd.grad(drop.dropout_add(x.float(), half, 0.5, seed=seed), half, dy)[0], dy.bfloat16())
    y = drop.dropout(x, 0.5, seed=seed)
    assert torch.equal(torch.func.vmap(lambda t: drop.dropout(t, 0.5, seed=seed))(x[None])[0], y)
    assert torch.equal(torch.compile(lambda t: drop.dropout(t, 0.5, seed=seed), backend="eager")(x), y)
    out, tangent = torch.func.jvp(lambda t: drop.dropout(t, 0.5, seed=seed), (x,), (x,))
    assert torch.equal(tangent, y)
    leaf = x.clone().requires_grad_()
    y = drop.dropout(leaf, 0.5, seed=seed)
    with pytest.raises(RuntimeError, match="batches of gradients"):
        torch.autograd.grad(y, leaf, torch.stack([y.detach()] * 2), is_grads_batched=True)


@pytest.mark.gpu
def test_elements_past_32_bits(gen):
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    n = (1 << 32) + 5
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = drop.dropout(x, 0.5, seed=torch.tensor([3, 4], device="cuda"))
    at = [0, 1, (1 << 31) + 1, (1 << 32) - 1, 1 << 32, n - 1]
    assert [bool(v) for v in y[at].tolist()] == [w >= 1 << 31 for w in _words(3, 4, at)]
