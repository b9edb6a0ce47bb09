"""Attention with a sliding window and first tokens that stay visible (`makani_b200/ops/attention.py`), and the way of a fused projection through norms,
rotation and attention (`makani_b200/ops/rotary.py`), against their definitions in 64 bits, sequence by sequence and head by head.

Tolerances as in `test_attention.py`, where they are derived: what a weight is off by does not depend on which weights there are."""

import math

import pytest
import torch

from makani_b200.ops import _ext
from makani_b200.ops import attention as attn
from makani_b200.ops import rotary as rot

B_STEP = 2.0 ** -8
F_STEP = 2.0 ** -19


def _seen(n, causal, window, sinks, device):
    """The definition, pair by pair of places."""
    i, j = torch.arange(n, device=device)[:, None], torch.arange(n, device=device)[None, :]
    seen = torch.ones(n, n, dtype=torch.bool, device=device)
    if window is not None:
        left, right = window if isinstance(window, tuple) else (window, window)
        left, right = (n if w is None else w for w in (left, right))
        seen = ((j >= i - left) & (j <= i + right)) | (j < sinks)
    return seen & (j <= i) if causal else seen


def _oracle(q, k, v, do, scale, bounds, **mask):
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    G = q.shape[1] // k.shape[1]
    names = ("o", "dq", "dk", "dv")
    out = {n: torch.zeros_like(t) for n, t in zip(names, (q, q, k, v))}
    off = {n: torch.zeros_like(t) for n, t in zip(names, (q, q, k, v))}
    for lo, hi in bounds:
        n = hi - lo
        for h in range(q.shape[1]) if n else ():
            qs, ks, vs, gs = q[lo:hi, h], k[lo:hi, h // G], v[lo:hi, h // G], do[lo:hi, h]
            s = (qs @ ks.mT * scale).masked_fill(~_seen(n, device=q.device, **mask), -math.inf)
            p = torch.softmax(s, -1)
            o = p @ vs
            e = F_STEP * (1 + 2 * (qs.abs() @ ks.abs().mT) * scale)
            dp = gs @ vs.mT
            delta = (gs * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            d = B_STEP * (gs * o).abs().sum(-1, keepdim=True) + F_STEP * (gs.abs() * o.abs()).sum(-1, keepdim=True)
            ds_off = B_STEP * ds.abs() + p * (d + e * (dp.abs() + delta.abs()) + F_STEP * (gs.abs() @ vs.abs().mT))
            out["o"][lo:hi, h], off["o"][lo:hi, h] = o, (p * (B_STEP + e)) @ vs.abs()
            out["dq"][lo:hi, h], off["dq"][lo:hi, h] = scale * ds @ ks, scale * (ds_off + F_STEP * ds.abs()) @ ks.abs()
            out["dk"][lo:hi, h // G] += scale * ds.mT @ qs
            off["dk"][lo:hi, h // G] += scale * (ds_off + F_STEP * ds.abs()).mT @ qs.abs()
            out["dv"][lo:hi, h // G] += p.mT @ gs
            off["dv"][lo:hi, h // G] += (p * (B_STEP + e)).mT @ gs.abs()
    return out, off


def _close(got, want, off, what):
    assert got.shape == want.shape and got.dtype == torch.bfloat16, what
    diff = (got.double() - want).abs()
    bound = off * (1 + B_STEP) + B_STEP * want.abs() + 1e-30
    bad = ~(diff <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((diff / bound).nan_to_num(9e9)[bad].max()):.2f} of the bound"


def _inputs(g, *lead, H, Hk, D):
    r = lambda h: torch.randn(*lead, h, D, device="cuda", generator=g).bfloat16()  # noqa: E731
    return r(H), r(Hk), r(Hk), r(H)


def _run(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = attn.attention(*leaves, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, leaves, do)))


def _check_batch(g, B, N, H, Hk, D, causal=False, window=None, sinks=0):
    q, k, v, do = _inputs(g, B, N, H=H, Hk=Hk, D=D)
    got = _run(q, k, v, do, causal=causal, window=window, sinks=sinks)
    for b in range(B):
        want, off = _oracle(q[b], k[b], v[b], do[b], D ** -0.5, [(0, N)], causal=causal, window=window, sinks=sinks)
        for n in want:
            _close(got[n][b], want[n], off[n], f"{n} of sample {b}")
    return got


def _check_packed(g, lens, H, Hk, D, behind=0, **mask):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    T = off[-1] + behind
    q, k, v, do = _inputs(g, T, H=H, Hk=Hk, D=D)
    for t in (q, k, v, do):      # what no sequence holds reaches nothing
        t[off[-1]:] = math.nan
    got = _run(q, k, v, do, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"), **mask)
    want, bound = _oracle(q[:off[-1]], k[:off[-1]], v[:off[-1]], do[:off[-1]], D ** -0.5, list(zip(off, off[1:])), **mask)
    for n in want:
        _close(got[n][:off[-1]], want[n], bound[n], n)
        assert not got[n][off[-1]:].any(), n


# ---------------------------------------------------------------------------------------------------- any machine

def test_refusals():
    q = torch.randn(2, 5, 4, 8)
    for bad in (-1, (1,), (1, 2, 3), (-1, 2), 1.5, True, (1, True), "3"):
        with pytest.raises(ValueError, match="window"):
            attn.attention(q, q, q, window=bad)
    for bad in (-1, 1.0, None, True):
        with pytest.raises(ValueError, match="sinks"):
            attn.attention(q, q, q, window=2, sinks=bad)
    with pytest.raises(ValueError, match="window"):
        attn.attention_qkv(torch.randn(2, 5, 96), 4, window=(2, -3))
    with pytest.raises(ValueError, match="sinks"):
        attn.attention_qkv(torch.randn(2, 5, 96), 4, sinks=-3)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (2, 0), ((3, 1), 2), ((None, 0), 0), ((1, None), 3), (100, 5), ((2, 2), 100)])
def test_cpu_formulation(causal, window, sinks, monkeypatch):
    torch.manual_seed(1)
    monkeypatch.setattr(attn, "QUERIES_AT_ONCE", 5)
    q, k, v, do = (torch.randn(17, h, 6, dtype=torch.float64) for h in (4, 2, 2, 4))
    mask = dict(causal=causal, window=window, sinks=sinks)
    for n in (1, 6, 17):
        assert torch.equal(attn.visible(n, **mask), _seen(n, device="cpu", **mask))
    bounds = [(0, 3), (3, 3), (3, 4), (4, 15)]
    want, _ = _oracle(q, k, v, do, 0.3, bounds, **mask)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = attn.attention(*leaves, scale=0.3, offsets=[0, 3, 3, 4, 15], **mask)
    for got, n in zip((o,) + torch.autograd.grad(o, leaves, do), ("o", "dq", "dk", "dv")):
        assert torch.allclose(got, want[n], atol=1e-12), n
    x = torch.cat([t.flatten(1) for t in (q, k, v)], 1)
    assert torch.allclose(attn.attention_qkv(x, 4, 2, scale=0.3, offsets=[0, 3, 3, 4, 15], **mask), want["o"], atol=1e-12)
    whole, _ = _oracle(q, k, v, do, 6 ** -0.5, [(0, 17)], **mask)
    assert torch.allclose(attn.attention_qkv(x[None], 4, 2, **mask)[0], whole["o"], atol=1e-12)
    same = torch.cat([q.flatten(1)] * 3, 1)
    want, _ = _oracle(q, q, q, do, 6 ** -0.5, [(0, 17)], **mask)
    assert torch.allclose(attn.attention_qkv(same[None], 4, **mask)[0], want["o"], atol=1e-12)


def test_gradient_formulas_against_differences():
    torch.manual_seed(2)
    q, k, v, do = (torch.randn(9, h, 5, dtype=torch.float64) for h in (4, 2, 2, 4))
    mask = dict(causal=False, window=(2, 1), sinks=1)
    want, _ = _oracle(q, k, v, do, 0.4, [(0, 2), (2, 9)], **mask)
    f = lambda *t: (_oracle(*t, do, 0.4, [(0, 2), (2, 9)], **mask)[0]["o"] * do).sum()  # noqa: E731
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn_like((q, k, v)[i])
        up, down = ([t + s * 1e-6 * d if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1))
        assert abs((f(*up) - f(*down)).item() / 2e-6 - (want[n] * d).sum().item()) < 1e-6


def test_path_on_the_cpu():
    """A fused projection through norms, rotation and attention is the three of them one after the other."""
    torch.manual_seed(3)
    axes = rot.RotaryAxes((4, 2), base=20.0)
    x = torch.randn(2, 9, 8 * 8, dtype=torch.float64, requires_grad=True)
    p = [torch.randn(8, dtype=torch.float64, requires_grad=True) for _ in range(4)]
    at = rot.grid_positions(3, 3)
    kw = dict(window=2, sinks=1)
    o = rot.rotary_attention_qkv(x, 4, 2, at, axes, *p, eps=1e-4, norm="rms", **kw)
    q, k, v = x.unflatten(-1, (8, 8)).split([4, 2, 2], 2)
    q, k = rot.norm_rotary_qk(q, k, p[0], p[1], at, axes, p[2], p[3], 1e-4, "rms")
    want = attn.attention(q, k, v, **kw)
    do = torch.randn_like(o)
    for a, b in zip(torch.autograd.grad(o, [x, *p], do), torch.autograd.grad(want, [x, *p], do)):
        assert torch.allclose(a, b, atol=1e-10)
    assert torch.allclose(o, want, atol=1e-12)
    assert torch.equal(rot.rotary_attention_qkv(x, 4, 2, **kw), attn.attention_qkv(x, 4, 2, **kw))


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
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D", [(2, 129, 4, 4, 8), (1, 700, 2, 1, 64), (1, 1111, 3, 3, 128), (3, 390, 4, 2, 40)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (40, 4), ((127, 128), 0), ((128, 0), 3), (300, 130), ((0, 200), 1), ((None, 10), 0), ((33, None), 260)])
def test_windows(gen, B, N, H, Hk, D, causal, window, sinks):
    _check_batch(gen, B, N, H, Hk, D, causal, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N", [1, 2, 127, 128, 129, 255, 256, 257, 383, 384, 385, 512, 640, 641])
@pytest.mark.parametrize("D", [64, 96])
def test_edges_of_tiles(gen, N, D, causal):
    for window in (1, 64, 127, 128, 129, (256, 255)):
        for sinks in (0, 1, 128, 129):
            _check_batch(gen, 1, N, 2, 1, D, causal, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hk,D,N,window,sinks", [(2, 2, 64, 6000, 200, 4), (4, 1, 128, 3001, 130, 200), (1, 1, 48, 9001, (500, 20), 1), (6, 2, 24, 4100, 60, 300),
                                                  (8, 8, 96, 2500, 300, 16), (1, 1, 64, 20000, 100, 1)])
def test_sinks_that_go_apart(gen, H, Hk, D, N, window, sinks, causal):
    """Long sequences, whose first keys have more queries than others: they are split over them and added up."""
    _check_batch(gen, 1, N, H, Hk, D, causal, window, sinks)


LENGTHS = [(300, 1, 0, 700, 64), (128, 256, 128, 0, 0, 129), (1,) * 40, (1500, 3, 900), (5, 0, 2200)]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("H,Hk,D,behind", [(4, 2, 64, 0), (3, 3, 128, 140), (2, 1, 40, 3)])
@pytest.mark.parametrize("window,sinks", [(70, 4), ((200, 10), 0), (16, 140)])
def test_packed_sequences(gen, lens, H, Hk, D, behind, causal, window, sinks):
    _check_packed(gen, lens, H, Hk, D, behind, causal=causal, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", [(1, 0, 0, 2, 0, 0, 3, 0), (0,) * 7 + (6,), (0, 0, 1), (137, 3) + (0,) * 142, (140, 3) + (0,) * 400, (0,) * 3000 + (1, 299)])
@pytest.mark.parametrize("H,Hk,D,behind", [(2, 1, 16, 0), (4, 2, 128, 5)])
@pytest.mark.parametrize("window,sinks", [(1, 1), ((2, 0), 0), (0, 300)])
def test_more_sequences_than_tokens(gen, lens, H, Hk, D, behind, window, sinks, causal):
    """Offsets with room for more sequences than there are, as a captured graph has them."""
    _check_packed(gen, lens, H, Hk, D, behind, causal=causal, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "rms"])
def test_path_with_more_sequences_than_tokens(gen, norm):
    """The fused calls: what the operators one after the other give."""
    off = torch.tensor([0, 1, 1, 1, 3, 3, 3, 6, 6], dtype=torch.int32, device="cuda")
    axes, at = rot.RotaryAxes((8, 8)), rot.grid_positions(2, 3, device="cuda")
    x = torch.randn(6, 8 * 16, device="cuda", generator=gen).bfloat16().requires_grad_()
    w = [torch.randn(16, device="cuda", generator=gen).requires_grad_() for _ in range(2)] if norm else [None] * 2
    kw, leaves = dict(offsets=off, window=1, sinks=1), [x] + [t for t in w if norm]
    q, k, v = x.unflatten(-1, (-1, 16)).split([4, 2, 2], -2)
    do = torch.randn(6, 4, 16, device="cuda", generator=gen).bfloat16()
    if norm:
        turned = rot.norm_rotary_qk(q, k, *w, at, axes, norm=norm)
    else:
        turned = rot.rotary_qk(q, k, at, axes)
    for got, want, of in ((rot.rotary_attention_qkv(x, 4, 2, at, axes, *w, norm=norm, **kw), attn.attention(*turned, v, **kw), leaves),
                          (attn.attention_qkv(x, 4, 2, **kw), attn.attention(q, k, v, **kw), [x])):
        assert torch.equal(got, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, of, do, retain_graph=True), torch.autograd.grad(want, of, do, retain_graph=True)))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_packed_sinks_that_go_apart(gen, causal):
    _check_packed(gen, (7000, 40, 1500), 4, 1, 64, 5, causal=causal, window=100, sinks=3)
    _check_packed(gen, (3001, 0, 2), 2, 2, 128, 77, causal=causal, window=(30, 60), sinks=131)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,H,Hk,window,sinks,causal", [(70001, 3, 1, 1, 1, 0, False), (66000, 4, 2, 1, (1, 1), 1, False), (70001, 5, 1, 1, 2, 0, True),
                                                          (1, 70, 70001, 70001, 3, 0, False), (2, 5, 33000, 16500, 1, 2, True)])
def test_many_sequences_and_heads(gen, B, N, H, Hk, window, sinks, causal):
    """More of either than a grid has along y."""
    q, k, v, do = _inputs(gen, B, N, H=H, Hk=Hk, D=8)
    mask = dict(causal=causal, window=window, sinks=sinks)
    got, G = _run(q, k, v, do, **mask), H // Hk
    for b in {0, 1, 65534, 65535, 65536, B - 1} & set(range(B)):
        for h in {0, 1, 65534, 65535, 65536, Hk - 1} & set(range(Hk)):
            at = (slice(h * G, (h + 1) * G), slice(h, h + 1), slice(h, h + 1), slice(h * G, (h + 1) * G))
            want, off = _oracle(*(t[b, :, a] for t, a in zip((q, k, v, do), at)), 8 ** -0.5, [(0, N)], **mask)
            for n, a in zip(want, (at[0], at[0], at[1], at[1])):
                _close(got[n][b, :, a], want[n], off[n], f"{n} of sample {b}, head {h}")


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D", [(32, 384, 8, 8, 64), (20, 440, 8, 2, 128), (160, 129, 1, 1, 24), (9, 1300, 8, 8, 48)])
def test_short_sequences_of_several_tiles(gen, B, N, H, Hk, D, causal):
    q, k, v, do = _inputs(gen, B, N, H=H, Hk=Hk, D=D)
    mask = dict(causal=causal, window=100, sinks=2)
    got = _run(q, k, v, do, **mask)
    for b in (0, B // 2, B - 1):
        want, off = _oracle(q[b], k[b], v[b], do[b], D ** -0.5, [(0, N)], **mask)
        for n in want:
            _close(got[n][b], want[n], off[n], f"{n} of sample {b}")


@pytest.mark.gpu
def test_windows_over_everything_are_none(gen):
    """The same bits as without one, on the same kernels."""
    q, k, v, do = _inputs(gen, 2, 500, H=4, Hk=2, D=64)
    for causal, windows in ((False, [499, (499, None), (None, None), 10 ** 9]), (True, [499, (None, 0), (499, 0), (10 ** 12, 3)])):
        want = _run(q, k, v, do, causal=causal)
        for window in windows:
            got = _run(q, k, v, do, causal=causal, window=window, sinks=3)
            assert all(torch.equal(got[n], want[n]) for n in want), (causal, window)


@pytest.mark.gpu
def test_hidden_scores_may_be_large(gen):
    """Scores that a window hides, far above those that are seen, leave no trace; nor do they where a row's sum is made again."""
    q, k, v, do = _inputs(gen, 1, 900, H=2, Hk=2, D=64)
    k[:, 500:520] *= 60
    mask = dict(causal=False, window=50, sinks=2)
    got = _run(q, k, v, do, **mask)
    want, off = _oracle(q[0], k[0], v[0], do[0], 0.125, [(0, 900)], **mask)
    for n in want:
        _close(got[n][0], want[n], off[n], n)
    k2, v2 = k.clone(), v.clone()
    k2[:, 500:520], v2[:, 500:520] = 30 * torch.randn_like(k2[:, 500:520]), 100.0
    other = _run(q, k2, v2, do, **mask)
    far = torch.arange(900, device="cuda")
    far = (far < 449) | (far > 570)
    assert torch.equal(other["o"][:, far], got["o"][:, far]) and torch.equal(other["dq"][:, far], got["dq"][:, far])


@pytest.mark.gpu
def test_strides_of_windows(gen):
    x = torch.randn(2, 300, 3, 4, 64, device="cuda", generator=gen).bfloat16()
    do = torch.randn(2, 300, 4, 64, device="cuda", generator=gen).bfloat16()
    dense = _run(*(x[:, :, i].contiguous() for i in range(3)), do, window=40, sinks=2)
    views = _run(*x.unbind(2), do.transpose(1, 2).contiguous().transpose(1, 2), window=40, sinks=2)
    assert all(torch.equal(dense[n], views[n]) for n in dense)
    flat = x.flatten(2).requires_grad_()
    o = attn.attention_qkv(flat, 4, window=40, sinks=2)
    g, = torch.autograd.grad(o, flat, do)
    assert torch.equal(o, dense["o"]) and torch.equal(g.view_as(x)[:, :, 1], dense["dk"])
    for D in (1, 20, 127):
        _check_batch(gen, 1, 200, 2, 1, D, False, 30, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [None, (5000, 30, 4000)])
def test_repeats_itself_and_replays(gen, lens):
    """The same bits every time, and captured graphs, two of them in turn, that replay with other tokens and lengths."""
    T = 9100
    q, k, v, do = _inputs(gen, *((1, T) if lens is None else (T,)), H=4, Hk=2, D=64)
    off = None if lens is None else torch.tensor([0, 5000, 5030, 9030], dtype=torch.int32, device="cuda")
    call = lambda: _run(q, k, v, do, causal=True, window=300, sinks=4, offsets=off)  # noqa: E731
    first, again = call(), call()
    assert all(torch.equal(first[n], again[n]) for n in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    with torch.cuda.stream(side):
        call()
        torch.cuda.synchronize()
        for g in graphs:
            with torch.cuda.graph(g, stream=side):
                outs.append(call())
    torch.cuda.synchronize()
    for g, out in zip(graphs, outs):
        q.copy_(torch.randn_like(q))
        if off is not None:
            off.copy_(torch.tensor([0, 17, 3000, 8000], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = call()
        assert all(torch.equal(out[n], want[n]) for n in want)


@pytest.mark.gpu
def test_window_offsets_out_of_range_are_clamped(gen):
    q, k, v, do = _inputs(gen, 600, H=2, Hk=2, D=64)
    want = _run(q, k, v, do, offsets=torch.tensor([0, 250, 600], dtype=torch.int32, device="cuda"), window=60, sinks=2)
    got = _run(q, k, v, do, offsets=torch.tensor([0, 250, 10 ** 6], dtype=torch.int32, device="cuda"), window=60, sinks=2)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "layer", "rms"])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("H,Hk,D,window", [(4, 2, 64, 90), (3, 3, 24, None), (8, 2, 128, (40, 70))])
def test_path(gen, norm, packed, H, Hk, D, window):
    """The fused projection's way in one call: the bits of the operators one after the other, and gradients of the projection and the norms."""
    N = 400
    lead = (N,) if packed else (2, N)
    axes = rot.RotaryAxes((D // 2, D // 4))
    at = rot.grid_positions(20, 20, device="cuda")
    off = torch.tensor([0, 150, 150, 380], dtype=torch.int32, device="cuda") if packed else None
    x = torch.randn(*lead, (H + 2 * Hk) * D, device="cuda", generator=gen).bfloat16().requires_grad_()
    p = [(0.2 * torch.randn(D, device="cuda", generator=gen) + (i < 2)).requires_grad_() for i in range(4)] if norm else [None] * 4
    leaves = [x] + [t for t in p if t is not None]
    kw = dict(offsets=off, window=window, sinks=3)
    o = rot.rotary_attention_qkv(x, H, Hk, at, axes, *p, norm=norm, **kw)
    q, k, v = x.unflatten(-1, (-1, D)).split([H, Hk, Hk], -2)
    q, k = rot.norm_rotary_qk(q, k, p[0], p[1], at, axes, p[2], p[3], norm=norm) if norm else rot.rotary_qk(q, k, at, axes)
    want = attn.attention(q, k, v, **kw)
    assert torch.equal(o, want)
    do = torch.randn(o.shape, device="cuda", generator=gen).bfloat16()
    for n, a, b in zip(["x", "qw", "kw", "qb", "kb"], torch.autograd.grad(o, leaves, do, retain_graph=True), torch.autograd.grad(want, leaves, do)):
        assert a.dtype == b.dtype and torch.equal(a, b), n
    if packed:      # what tokens of no sequence hold reaches nothing
        with torch.no_grad():
            bad = x.detach().clone()
            bad[380:] = math.nan
        bad.requires_grad_()
        other = rot.rotary_attention_qkv(bad, H, Hk, at, axes, *p, norm=norm, **kw)
        assert torch.equal(other, o)
        for a, b in zip(torch.autograd.grad(other, [bad, *leaves[1:]], do), torch.autograd.grad(o, leaves, do)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [None, "layer", "rms"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("D,bands,inter", [(64, (32, 16), False), (24, (12, 12), False), (40, (10, 6), False), (128, (64, 64), True)])
def test_positions_behind_the_last_sequence_reach_nothing(gen, D, bands, inter, value, norm):
    """The same bits whatever positions the tokens of no sequence have."""
    axes = rot.RotaryAxes(bands, interleaved=inter)
    off = torch.tensor([0, 150, 150, 333], dtype=torch.int32, device="cuda")
    x = torch.randn(400, 8 * D, device="cuda", generator=gen).bfloat16().requires_grad_()
    p = [(0.2 * torch.randn(D, device="cuda", generator=gen) + (i < 2)).requires_grad_() for i in range(4)] if norm else [None] * 4
    do = torch.randn(400, 4, D, device="cuda", generator=gen).bfloat16()
    at = 100 * torch.rand(400, 2, device="cuda", generator=gen)
    bad = at.clone()
    bad[333:] = value

    def call(at):
        o = rot.rotary_attention_qkv(x, 4, 2, at, axes, *p, norm=norm, offsets=off, window=50, sinks=1)
        return [o, *torch.autograd.grad(o, [x] + [t for t in p if t is not None], do)]

    for got, want in zip(call(bad), call(at)):
        assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.gpu
def test_transforms_and_refusals_of_windows(gen):
    q, k, v, do = _inputs(gen, 2, 60, H=2, Hk=1, D=16)
    mask = dict(window=9, sinks=1)
    o = attn.attention(q, k, v, **mask)
    many = torch.func.vmap(lambda a, b, c: attn.attention(a[None], b[None], c[None], **mask)[0])(q, k, v)
    assert torch.allclose(many.float(), o.float(), atol=0.03)
    leaf = q.clone().requires_grad_()
    y = attn.attention(leaf, k, v, **mask)
    with pytest.raises(RuntimeError, match="batches of gradients"):
        torch.autograd.grad(y, leaf, torch.stack([do] * 2), is_grads_batched=True)
    x = torch.randn(2, 60, 64, device="cuda", generator=gen).bfloat16()
    axes, at = rot.RotaryAxes((8,)), torch.arange(60, device="cuda")[:, None]
    o = rot.rotary_attention_qkv(x, 2, 1, at, axes, **mask)
    many = torch.func.vmap(lambda t: rot.rotary_attention_qkv(t[None], 2, 1, at, axes, **mask)[0])(x)
    assert torch.allclose(many.float(), o.float(), atol=0.03)
    with pytest.raises(RuntimeError, match="sinks"):
        _ext.require().attention(q, k, v, None, False, 0.25, 4, 4, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("N,H,Hk,D,window,sinks", [(4100, 6, 2, 24, 60, 300), (2177, 4, 4, 64, 40, 0), (1030, 8, 1, 8, 129, 3), (2052, 3, 3, 96, 20, 1)])
def test_last_tiles_of_few_keys_repeat_themselves(gen, N, H, Hk, D, window, sinks, causal):
    """Warps whose columns nobody sees are through with a tile before the others, and must not run into the next but one: the same bits, many times over."""
    q, k, v, do = _inputs(gen, 1, N, H=H, Hk=Hk, D=D)
    mask = dict(causal=causal, window=window, sinks=sinks)
    first = _run(q, k, v, do, **mask)
    want, off = _oracle(q[0], k[0], v[0], do[0], D ** -0.5, [(0, N)], **mask)
    for n in want:
        _close(first[n][0], want[n], off[n], n)
    for _ in range(150):
        again = _run(q, k, v, do, **mask)
        assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 96])
def test_nan_of_a_neighbour_stays_there(gen, D, causal):
    """Sequences side by side in tiles: what one holds, NaN too, reaches no other, through window and sinks, forward and backward."""
    off = [0, 200, 201, 700, 1000]
    q, k, v, do = _inputs(gen, 1000, H=4, Hk=2, D=D)
    kw = dict(offsets=torch.tensor(off, dtype=torch.int32, device="cuda"), causal=causal, window=70, sinks=3)
    want = _run(q, k, v, do, **kw)
    for i in (1, 2):
        bad = [t.clone() for t in (q, k, v, do)]
        for t in bad:
            t[off[i]:off[i + 1]] = math.nan
        got = _run(*bad, **kw)
        for n in want:
            for lo, hi in ((0, off[i]), (off[i + 1], 1000)):
                assert torch.equal(got[n][lo:hi], want[n][lo:hi]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_other_types_through_torch(gen, dtype):
    q, k, v, do = (t.to(dtype) for t in _inputs(gen, 300, H=4, Hk=2, D=24))
    off = [0, 120, 120, 290]
    for causal in (False, True):
        mask = dict(causal=causal, window=(30, 10), sinks=2)
        got = _run(q, k, v, do, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"), **mask)
        want, _ = _oracle(q, k, v, do, 24 ** -0.5, list(zip(off, off[1:])), **mask)
        for n in want:
            assert torch.allclose(got[n].double(), want[n], atol=2e-5 if dtype == torch.float32 else 2e-2), n
    rot.rotary(q.float(), torch.arange(300, device="cuda")[:, None], rot.RotaryAxes((24,)))      # (one call on a kernel)


@pytest.mark.gpu
def test_two_streams_at_once(gen):
    """Two calls at the same time, each with workspaces of its own."""
    sets = [_inputs(gen, 1, 5000, H=4, Hk=1, D=64) for _ in range(2)]
    mask = dict(causal=True, window=200, sinks=4)
    want = [_run(*s, **mask) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _run(*sets[i], **mask)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[n], b[n]) for n in b)
