"""Softmax attention (`makani_b200/ops/attention.py`) against its definition in 64 bits, sequence by sequence and head by head.

Tolerances, element by element.  Half a step of bf16 is B = 2^-8 relative (`eps / 2`); fp32 sums and the special function's 2^x (two steps of
2^-23) are counted as F = 2^-19 of the sum of magnitudes.  A score is off by at most F times sum |q k| scale, a weight P then by P (F + that).

    o  = sum P v          P is rounded to bf16:     |o|  off by  (B + e) sum P |v|,   then rounded once
    dS = P (dP - delta)   delta holds the rounded o and do: off by d = B sum |do o|;    dS is rounded to bf16
    dq = scale sum dS k   off by  scale sum (B |dS| + P (d + e (|dP| + |delta|) + F sum|do v|)) |k|,  then rounded once
    dk the same over the queries; dv = sum P do  off by  (B + e) sum P |do|."""

import math
import os
import subprocess
import sys

import pytest
import torch

from makani_b200.ops import _ext
from makani_b200.ops import attention as attn

B_STEP = 2.0 ** -8
F_STEP = 2.0 ** -19


def _oracle(q, k, v, do, causal, scale, bounds, o_low=None):
    """64-bit outputs and bounds of [N, H, D] tensors; `bounds`: sequences.  Rows of no sequence are zero."""
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    G = q.shape[1] // k.shape[1]
    names = ("o", "dq", "dk", "dv")
    out = {n: torch.zeros_like(t) for n, t in zip(names, (q, q, k, v))}
    off = {n: torch.zeros_like(t) for n, t in zip(names, (q, q, k, v))}
    for lo, hi in bounds:
        n = hi - lo
        for h in range(q.shape[1]) if n else ():
            qs, ks, vs, gs = q[lo:hi, h], k[lo:hi, h // G], v[lo:hi, h // G], do[lo:hi, h]
            s = qs @ ks.mT * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=s.device).triu(1), -math.inf)
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


def _inputs(g, *lead, H, Hk, D, amp=1.0):
    r = lambda h: torch.randn(*lead, h, D, device="cuda", generator=g)  # noqa: E731
    return (amp * r(H)).bfloat16(), (amp * r(Hk)).bfloat16(), r(Hk).bfloat16(), r(H).bfloat16()


def _run(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = attn.attention(*leaves, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(),) + torch.autograd.grad(o, leaves, do)))


def _check_batch(g, B, N, H, Hk, D, causal, scale=None, amp=1.0):
    q, k, v, do = _inputs(g, B, N, H=H, Hk=Hk, D=D, amp=amp)
    got = _run(q, k, v, do, causal=causal, scale=scale)
    torch.cuda.synchronize()
    _ext.check_device_errors()
    for b in range(B):
        want, off = _oracle(q[b], k[b], v[b], do[b], causal, scale or D ** -0.5, [(0, N)])
        for n in want:
            _close(got[n][b], want[n], off[n], f"{n} of sample {b}")


# ---------------------------------------------------------------------------------------------------- any machine

def test_refusals():
    q, k = torch.randn(2, 5, 4, 8), torch.randn(2, 5, 2, 8)
    for bad in ((q, k, k[:, :4]), (q, k[:, :4], k[:, :4]), (q, k[:1], k[:1]), (q, k[..., :4], k[..., :4]), (q, k.double(), k.double()), (q[0], k[0], k[0])):
        with pytest.raises(ValueError):
            attn.attention(*bad)
    with pytest.raises(ValueError, match="divide"):
        attn.attention(q[:, :, :3], k, k)
    for s in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            attn.attention(q, k, k, scale=s)
    with pytest.raises(ValueError, match="offsets"):
        attn.attention(q, k, k, offsets=torch.tensor([0, 5]))
    for off in ([0, 6], [1, 5], [0, 3, 2], [[0, 5]], [0.0, 5.0]):
        with pytest.raises(ValueError, match="offsets"):
            attn.attention(q[0], k[0], k[0], offsets=torch.tensor(off))
    x = torch.randn(2, 5, 64)
    with pytest.raises(ValueError, match="divide"):
        attn.attention_qkv(x, 4, 3)
    with pytest.raises(ValueError, match="channels"):
        attn.attention_qkv(x, 5)
    with pytest.raises(ValueError):
        attn.attention_qkv(x[0], 4, 2)
    with pytest.raises(ValueError, match="offsets"):
        attn.attention_qkv(x[0], 4, 2, offsets=torch.tensor([0, 9]))


@pytest.mark.parametrize("causal", [False, True])
def test_cpu_formulation(causal):
    torch.manual_seed(1)
    q, k, v, do = (torch.randn(11, h, 6, dtype=torch.float64) for h in (4, 2, 2, 4))
    bounds = [(0, 3), (3, 3), (3, 4), (4, 9)]
    want, _ = _oracle(q, k, v, do, causal, 0.3, bounds)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = attn.attention(*leaves, causal=causal, scale=0.3, offsets=[0, 3, 3, 4, 9])
    for got, n in zip((o,) + torch.autograd.grad(o, leaves, do), ("o", "dq", "dk", "dv")):
        assert torch.allclose(got, want[n], atol=1e-12), n
    x = torch.cat([t.flatten(1) for t in (q, k, v)], 1)
    assert torch.allclose(attn.attention_qkv(x, 4, 2, causal, 0.3, [0, 3, 3, 4, 9]), want["o"], atol=1e-12)
    whole, _ = _oracle(q, k, v, do, causal, 6 ** -0.5, [(0, 11)])
    assert torch.allclose(attn.attention(q[None], k[None], v[None], causal)[0], whole["o"], atol=1e-12)
    assert torch.allclose(attn.attention_qkv(x[None], 4, 2, causal)[0], whole["o"], atol=1e-12)


def test_gradient_formulas_against_differences():
    torch.manual_seed(2)
    q, k, v, do = (torch.randn(7, h, 5, dtype=torch.float64) for h in (4, 2, 2, 4))
    want, _ = _oracle(q, k, v, do, True, 0.4, [(0, 2), (2, 7)])
    f = lambda *t: (_oracle(*t, do, True, 0.4, [(0, 2), (2, 7)])[0]["o"] * do).sum()  # noqa: E731
    h = 1e-6
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn_like((q, k, v)[i])
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1))
        assert abs(float((want[n] * d).sum() - (f(*up) - f(*down)) / (2 * h))) < 1e-7, n


# ---------------------------------------------------------------------------------------------------- the kernels

@pytest.fixture
def gen():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.available()
    return torch.Generator("cuda").manual_seed(21)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D", [
    (1, 1, 1, 1, 8), (2, 2, 2, 1, 16), (1, 127, 2, 2, 64), (3, 128, 2, 2, 48), (1, 129, 1, 1, 128), (2, 255, 2, 2, 64), (1, 256, 3, 1, 72),
    (1, 257, 4, 2, 64), (2, 384, 1, 1, 40), (1, 385, 2, 1, 128), (1, 1000, 4, 4, 24), (1, 641, 6, 2, 96), (2, 130, 12, 4, 112), (1, 2050, 2, 2, 56)])
def test_lengths_heads_and_widths(gen, B, N, H, Hk, D, causal):
    _check_batch(gen, B, N, H, Hk, D, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,H,Hk,D", [(1, 2500, 1, 1, 128), (2, 3001, 3, 1, 72), (1, 4096, 2, 2, 64), (1, 2305, 5, 5, 8), (3, 1921, 2, 2, 48)])
def test_few_rows_and_long_keys(gen, B, N, H, Hk, D):
    """What does not fill the SMs is split over the keys and joined."""
    _check_batch(gen, B, N, H, Hk, D, False)
    q, k, v, _ = _inputs(gen, B, N, H=H, Hk=Hk, D=D)
    k = (k.float() * torch.linspace(0.1, 12, N, device="cuda")[None, :, None, None]).bfloat16()      # parts of very different maxima
    with torch.no_grad():
        o = attn.attention(q, k, v)
    want, off = _oracle(q[0], k[0], v[0], torch.zeros_like(q[0]), False, D ** -0.5, [(0, N)])
    _close(o[0], want["o"], off["o"], "o")


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,H,Hk,D", [(1, 2700, 8, 8, 64), (1, 2561, 8, 2, 128), (2, 1700, 6, 1, 48), (1, 5003, 4, 4, 104)])
def test_last_wave_of_the_gradients(gen, B, N, H, Hk, D):
    """Tiles of queries and keys behind the last whole wave are split along the other axis (over the heads that share keys, too) and summed; twice, the same bits."""
    _check_batch(gen, B, N, H, Hk, D, False)
    q, k, v, do = _inputs(gen, B, N, H=H, Hk=Hk, D=D)
    first, again = _run(q, k, v, do), _run(q, k, v, do)
    assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hk,D", [(8, 2, 64), (8, 1, 128), (6, 2, 24), (12, 1, 96)])
def test_shared_heads_apart(gen, H, Hk, D):
    """Gradients of keys and values with few CTAs: the heads that share them in CTAs of their own, causal and in packed sequences among NaN."""
    _check_batch(gen, 1, 1100, H, Hk, D, True)
    at = [0, 700, 700, 701, 1630]
    for causal in (False, True):
        q, k, v, do = _inputs(gen, 1700, H=H, Hk=Hk, D=D)
        for x in (q, k, v, do):
            x[at[-1]:] = float("nan")
        got = _run(q, k, v, do, causal=causal, offsets=torch.tensor(at, dtype=torch.int32, device="cuda"))
        want, off = _oracle(q, k, v, do, causal, D ** -0.5, list(zip(at, at[1:])))
        for n in want:
            _close(got[n], want[n], off[n], n)
            assert not got[n][at[-1]:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [1, 5, 20, 65, 127])
def test_widths_that_are_padded(gen, D):
    _check_batch(gen, 1, 200, 2, 1, D, True)


@pytest.mark.gpu
def test_sharp_scores(gen):
    """Scores of some hundred: one weight of a row is nearly all of it, and maxima grow along the keys."""
    _check_batch(gen, 1, 700, 2, 2, 64, False, amp=4.0)
    q, k, v, do = _inputs(gen, 1, 900, H=2, Hk=2, D=64)
    k = (k.float() * torch.linspace(0.1, 12, 900, device="cuda")[None, :, None, None]).bfloat16()
    got = _run(q, k, v, do)
    want, off = _oracle(q[0], k[0], v[0], do[0], False, 0.125, [(0, 900)])
    for n in want:
        _close(got[n][0], want[n], off[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.02, 0.7])
def test_scale(gen, scale):
    _check_batch(gen, 1, 300, 2, 1, 48, False, scale=scale)


LENGTHS = [[5], [0], [1, 1, 1], [128, 128], [0, 130, 0, 257, 1, 0], [64, 300, 63, 1, 129], [31] * 40 + [0] * 30 + [2] * 9, [512, 3, 700]]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("H,Hk,D,behind", [(4, 2, 64, 0), (3, 3, 128, 140), (2, 1, 40, 3)])
def test_packed_sequences(gen, lens, H, Hk, D, behind, causal):
    """Neighbours hold NaN and infinities in their turn: nothing of them may reach a sequence."""
    T = sum(lens) + behind
    if T == 0:
        T = behind = 1
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    bounds = list(zip(at, at[1:]))
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    q, k, v, do = _inputs(gen, T, H=H, Hk=Hk, D=D)
    for t in (q, k, v, do):
        t[at[-1]:] = float("nan")
    got = _run(q, k, v, do, causal=causal, offsets=offsets)
    torch.cuda.synchronize()
    _ext.check_device_errors()
    want, off = _oracle(q, k, v, do, causal, D ** -0.5, bounds)
    for n in want:
        _close(got[n], want[n], off[n], n)
        assert not got[n][at[-1]:].any()
    whole = max(range(len(lens)), key=lambda i: lens[i])
    dirty = [t.clone() for t in (q, k, v, do)]
    keep = torch.zeros(T, dtype=torch.bool, device="cuda")
    keep[at[whole]:at[whole + 1]] = True
    for t, bad in zip(dirty, (float("nan"), float("inf"), float("nan"), float("-inf"))):
        t[~keep] = bad
    again = _run(*dirty, causal=causal, offsets=offsets)
    for n in want:
        assert torch.equal(again[n][keep], got[n][keep]), n


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_fused_projection(gen, packed):
    """The same bits as separate tensors; the gradient of the projection's output in one tensor."""
    H, Hk, D = 6, 2, 48
    lead = (500,) if packed else (2, 250)
    kw = dict(causal=True, offsets=torch.tensor([0, 200, 200, 490], dtype=torch.int32, device="cuda") if packed else None)
    x = torch.randn(*lead, (H + 2 * Hk) * D, device="cuda", generator=gen).bfloat16().requires_grad_()
    do = torch.randn(*lead, H, D, device="cuda", generator=gen).bfloat16()
    o = attn.attention_qkv(x, H, Hk, **kw)
    dx = torch.autograd.grad(o, x, do)[0]
    q, k, v = x.detach().unflatten(-1, (-1, D)).split([H, Hk, Hk], -2)
    got = _run(q, k, v, do, **kw)
    assert torch.equal(o, got["o"]) and torch.equal(dx, torch.cat([got[n].flatten(-2) for n in ("dq", "dk", "dv")], -1))


@pytest.mark.gpu
def test_strides(gen):
    """Views of other layouts give the bits of dense tensors."""
    B, N, H, D = 2, 150, 4, 32
    q, k, v, do = _inputs(gen, B, N, H=H, Hk=H, D=D)
    want = _run(q, k, v, do, causal=True)

    def same(*views, g=do):
        got = _run(*views, g, causal=True)
        assert all(torch.equal(got[n], want[n]) for n in want)

    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    same(*heads_first, g=do.transpose(1, 2).contiguous().transpose(1, 2))
    same(*(t.repeat(1, 1, 1, 2).view(B, N, H, 2, D)[..., 0, :] for t in (q, k, v)))
    same(*(torch.cat([t, t[..., :1]], -1)[..., :D] for t in (q, k, v)))              # rows off a 16-byte boundary
    same(*(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (q, k, v)))
    same(*(t.transpose(0, 3).contiguous().transpose(0, 3) for t in (q, k, v)))
    # one head's keys and values, seen by all (stride 0): the gradients of the views add up to that of the head
    one = _run(q, k[:, :, :1].expand(B, N, H, D), v[:, :, :1].expand(B, N, H, D), do)
    two = _run(q, k[:, :, :1].repeat(1, 1, H, 1), v[:, :, :1].repeat(1, 1, H, 1), do)
    assert all(torch.equal(one[n], two[n]) for n in one)
    grad = _run(q, k, v, do[:, :, :1, :1].expand(B, N, H, D))
    full = _run(q, k, v, do[:, :, :1, :1].expand(B, N, H, D).contiguous())
    assert all(torch.equal(grad[n], full[n]) for n in full)


@pytest.mark.gpu
def test_empty_and_partial_gradients(gen):
    q, k, v, do = _inputs(gen, 2, 0, H=2, Hk=2, D=16)
    got = _run(q, k, v, do)
    assert all(t.numel() == 0 for t in got.values())
    q, k, v, do = _inputs(gen, 2, 140, H=2, Hk=2, D=16)
    want = _run(q, k, v, do)
    kl = k.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(attn.attention(q, kl, v), kl, do)[0], want["dk"])
    with torch.no_grad():
        assert torch.equal(attn.attention(q, kl, v), want["o"])
    ql = q.clone().requires_grad_()
    dq = torch.autograd.grad(attn.attention(ql, k, v), ql, do, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivatives"):
        dq.float().sum().backward()


@pytest.mark.gpu
def test_rows_that_overflow_stay_alone(gen):
    """A query with NaN and one with infinities spoil their own rows of the output and nothing else."""
    q, k, v, do = _inputs(gen, 1, 300, H=2, Hk=2, D=32)
    clean = attn.attention(q, k, v)
    q[0, 7, 0, 3], q[0, 200, 1, 0] = float("nan"), float("inf")
    o = attn.attention(q, k, v)
    assert o[0, 7, 0].isnan().all() and o[0, 200, 1].isnan().all()
    keep = torch.ones(300, 2, dtype=torch.bool, device="cuda")
    keep[7, 0] = keep[200, 1] = False
    assert torch.equal(o[0][keep], clean[0][keep])


@pytest.mark.gpu
def test_repeats_itself_and_replays(gen):
    """The same bits again, on another stream beside other work, and from a captured graph that reads new inputs and offsets."""
    q, k, v, do = _inputs(gen, 900, H=4, Hk=2, D=64)
    offsets = torch.tensor([0, 100, 700, 900], dtype=torch.int32, device="cuda")
    first = _run(q, k, v, do, causal=True, offsets=offsets)
    same = lambda a, b: all(torch.equal(a[n], b[n]) for n in a)  # noqa: E731
    assert same(first, _run(q, k, v, do, causal=True, offsets=offsets))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = _run(q, k, v, do, causal=True, offsets=offsets)
        held = [t.clone() for t in (q, k, v, do, offsets)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = _run(*held[:4], causal=True, offsets=held[4])
    assert same(first, _run(q, k, v, do, causal=True, offsets=offsets))
    torch.cuda.current_stream().wait_stream(side)
    assert same(first, beside)
    for new in ([0, 100, 700, 900], [0, 300, 300, 890]):
        held[4].copy_(torch.tensor(new, dtype=torch.int32))
        held[0].copy_(q.flip(0))
        graph.replay()
        assert same(got, _run(q.flip(0), k, v, do, causal=True, offsets=held[4].clone()))
    del graph


@pytest.mark.gpu
def test_offsets_out_of_range_are_clamped(gen):
    q, k, v, do = _inputs(gen, 300, H=2, Hk=1, D=64)
    far = _run(q, k, v, do, offsets=torch.tensor([0, 120, 100000], dtype=torch.int32, device="cuda"))
    want = _run(q, k, v, do, offsets=torch.tensor([0, 120, 300], dtype=torch.int32, device="cuda"))
    assert all(torch.equal(far[n], want[n]) for n in want)
    long = _run(q, k, v, do, offsets=torch.tensor([0, 120, 300], device="cuda"))       # int64, and from the host
    host = _run(q, k, v, do, offsets=[0, 120, 300])
    assert all(torch.equal(long[n], want[n]) and torch.equal(host[n], want[n]) for n in want)


@pytest.mark.gpu
def test_refusals_on_the_device(gen):
    q, k, v, _ = _inputs(gen, 4, H=2, Hk=1, D=64)
    with pytest.raises(ValueError, match="offsets"):
        attn.attention(q, k, v, offsets=torch.tensor([0.0, 4.0], device="cuda"))
    with pytest.raises(ValueError, match="device"):
        attn.attention(q, k.cpu(), v.cpu(), offsets=[0, 4])


@pytest.mark.gpu
def test_gradient_against_differences(gen):
    """Steps of the kernel's own outputs along its gradient.  Outputs are bf16: the difference is known to the sum of their half steps."""
    N, H, D, h = 200, 2, 32, 2.0 ** -3
    q, k, v, do = _inputs(gen, 1, N, H=H, Hk=H, D=D)
    got = _run(q, k, v, do)
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn(q.shape, device="cuda", generator=gen)
        up, down = ([(t.float() + s * h * d).bfloat16() if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1))
        moved = up[i].double() - down[i].double()
        f = [(attn.attention(*t).double() * do.double()).sum() for t in (up, down)]
        ref = [_oracle(*(x[0] for x in t), do[0], False, D ** -0.5, [(0, N)]) for t in (up, down)]
        left_out = sum(s * (r[0]["o"] * do[0].double()).sum() for s, r in zip((1, -1), ref)) - \
            (_oracle(q[0], k[0], v[0], do[0], False, D ** -0.5, [(0, N)])[0][n] * moved[0]).sum()
        off = sum(((r[1]["o"] * (1 + B_STEP) + B_STEP * r[0]["o"].abs()) * do[0].double().abs()).sum() for r in ref)
        own = _oracle(q[0], k[0], v[0], do[0], False, D ** -0.5, [(0, N)])
        off = off + ((own[1][n] * (1 + B_STEP) + B_STEP * own[0][n].abs()) * moved[0].abs()).sum()
        assert abs(float(f[0] - f[1] - left_out - (got[n].double() * moved).sum())) <= float(off), n


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [32, 96])
def test_nan_of_a_query_reaches_what_it_sees(gen, D, causal):
    """A query with NaN or infinity makes NaN of the gradients of all keys and values that it sees, wherever in a tile it stands, and changes no value's that it
    does not see."""
    N, first = 300, 136
    q, k, v, do = _inputs(gen, 16, N, H=2, Hk=2, D=D)
    clean = _run(q, k, v, do, causal=causal)
    dirty = q.clone()
    for b in range(16):
        dirty[b, first + b, 0, 3] = float("nan") if b < 8 else float("inf")
    got = _run(dirty, k, v, do, causal=causal)
    for b in range(16):
        seen = first + b + 1 if causal else N
        assert got["dq"][b, first + b, 0].isnan().all() and got["o"][b, first + b, 0].isnan().all(), b
        for n in ("dk", "dv"):
            assert got[n][b, :seen, 0].isnan().all(), (n, b)
        assert torch.equal(got["dv"][b, seen:, 0], clean["dv"][b, seen:, 0]), b
    assert all(torch.equal(got[n][:, :, 1], clean[n][:, :, 1]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,H,D", [(2, 1, 4, 8), (1, 70, 2, 16), (2, 40, 1, 16), (1, 1, 3, 24), (3, 1, 1, 64), (1, 1, 1, 8)])
def test_strides_of_single_dimensions(gen, B, N, H, D):
    """A dimension of size one may have any stride: torch calls such a tensor contiguous."""
    q, k, v, do = _inputs(gen, B, N, H=H, Hk=H, D=D)
    want = _run(q, k, v, do)
    for odd in (1, 3, 8, 1 << 40):
        views = [t.as_strided(t.shape, [s if n > 1 else odd for n, s in zip(t.shape, t.stride())]) for t in (q, k, v, do)]
        got = _run(*views)
        assert all(torch.equal(got[n], want[n]) for n in want), odd
    x = torch.cat([t.flatten(2) for t in (q, k, v)], -1)
    y = x.as_strided(x.shape, [s if n > 1 else 1 for n, s in zip(x.shape, x.stride())]).requires_grad_()
    o = attn.attention_qkv(y, H)
    assert torch.equal(o, want["o"])
    dx = torch.autograd.grad(o, y, do)[0]
    assert torch.equal(dx, torch.cat([want[n].flatten(2) for n in ("dq", "dk", "dv")], -1))


@pytest.mark.gpu
def test_single_token_of_a_permuted_tensor(gen):
    t = torch.randn(2, 4, 8, 1, device="cuda", generator=gen).bfloat16()
    q = t.permute(0, 3, 1, 2)
    assert q.is_contiguous() and q.stride(1) == 1
    assert torch.equal(attn.attention(q, q, q), q)          # one key: its weight is 1


@pytest.mark.parametrize("packed", [False, True])
def test_no_query_heads(packed):
    """Refused: nothing attends, and torch's operator ends the process on a CPU."""
    lead, kw = ((10,), dict(offsets=[0, 4, 10])) if packed else ((2, 5), {})
    q, k = torch.randn(*lead, 0, 16), torch.randn(*lead, 2, 16)
    for dtype in (torch.float32, torch.bfloat16):
        with pytest.raises(ValueError, match="heads"):
            attn.attention(q.to(dtype), k.to(dtype), k.to(dtype), **kw)


@pytest.mark.gpu
def test_no_query_heads_in_the_extension(gen):
    q, k, _, _ = _inputs(gen, 2, 5, H=0, Hk=2, D=16)
    with pytest.raises(ValueError, match="heads"):
        attn.attention(q, k, k)
    with pytest.raises(RuntimeError, match="heads"):
        _ext.require().attention(q, k, k, None, False, 0.25)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offsets", [[0], [0, 0], [0, 0, 0]])
def test_tokens_of_no_sequence_only(dev, offsets, dtype):
    """Nothing but tokens behind the last sequence: outputs and all gradients are zero."""
    if dev == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    q, k, v = (torch.full((7, h, 16), float("nan"), device=dev, dtype=dtype, requires_grad=True) for h in (4, 2, 2))
    o = attn.attention(q, k, v, offsets=offsets)
    assert o.shape == q.shape and not o.any()
    for d, t in zip(torch.autograd.grad(o, (q, k, v), torch.ones_like(o)), (q, k, v)):
        assert d.shape == t.shape and not d.any()


@pytest.mark.gpu
def test_transforms_see_through_attention(gen):
    """vmap, tracing, compilation and fake tensors go by torch's operations.  Outputs are bf16 of either side: two roundings of weights and of the result."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    q, k, v, _ = _inputs(gen, 3, 20, H=2, Hk=1, D=16)
    other = _inputs(gen, 3, 20, H=2, Hk=1, D=16)[:3]
    own = lambda q, k, v: attn.attention(q, k, v, causal=True)  # noqa: E731
    near = lambda p, t: float((p.double() - t.double()).norm() / t.double().norm()) < 4 * B_STEP  # noqa: E731
    want = own(q, k, v)
    assert near(torch.func.vmap(lambda *t: own(*(x[None] for x in t))[0])(q, k, v), want)
    traced = torch.jit.trace(own, (q, k, v))
    assert near(traced(*other), own(*other))
    assert near(torch.compile(own, backend="eager", fullgraph=True)(*other), own(*other))
    x = torch.cat([t.flatten(2) for t in (q, k, v)], -1)
    traced = torch.jit.trace(lambda t: attn.attention_qkv(t, 2, 1, True), (x,))
    assert near(traced(x.flip(0)), attn.attention_qkv(x.flip(0), 2, 1, True))
    with FakeTensorMode() as mode:
        y = own(*(mode.from_tensor(t) for t in (q, k, v)))
    assert y.shape == q.shape


# What `one_tile_pays` gives to the forward kernels of one query tile (more pairs of tiles than SMs, short sequences), with several tiles of keys
@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,N,H,Hk,D", [(32, 384, 8, 8, 64), (20, 440, 8, 2, 128), (16, 768, 8, 4, 48), (27, 257, 6, 6, 72), (160, 129, 1, 1, 24)])
def test_short_sequences_of_several_tiles(gen, B, N, H, Hk, D, causal):
    q, k, v, do = _inputs(gen, B, N, H=H, Hk=Hk, D=D)
    k = (k.float() * torch.linspace(0.3, 3, N, device="cuda")[None, :, None, None]).bfloat16()      # maxima grow along the keys
    got = _run(q, k, v, do, causal=causal)
    torch.cuda.synchronize()
    _ext.check_device_errors()
    for b in (0, 1, B // 2, B - 1):
        want, off = _oracle(q[b], k[b], v[b], do[b], causal, D ** -0.5, [(0, N)])
        for n in want:
            _close(got[n][b], want[n], off[n], f"{n} of sample {b}")
    alone = _run(*(t[:1] for t in (q, k, v, do)), causal=causal)                   # few CTAs: another kernel, the same rows but for the order of sums
    want, off = _oracle(q[0], k[0], v[0], do[0], causal, D ** -0.5, [(0, N)])
    for n in want:
        _close(alone[n][0], want[n], off[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,Hk,D", [(8, 8, 64), (6, 2, 96), (8, 4, 40)])
def test_many_packed_sequences_of_several_tiles(gen, H, Hk, D, causal):
    lens = [130 + (97 * i) % 271 for i in range(40)] + [0, 1, 400]
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    T = at[-1] + 77
    q, k, v, do = _inputs(gen, T, H=H, Hk=Hk, D=D)
    for t in (q, k, v, do):
        t[at[-1]:] = float("nan")
    offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    got = _run(q, k, v, do, causal=causal, offsets=offsets)
    torch.cuda.synchronize()
    _ext.check_device_errors()
    want, off = _oracle(q, k, v, do, causal, D ** -0.5, list(zip(at, at[1:])))
    for n in want:
        _close(got[n], want[n], off[n], n)
        assert not got[n][at[-1]:].any()
    keep = torch.zeros(T, dtype=torch.bool, device="cuda")
    for i in range(0, len(lens), 2):
        keep[at[i]:at[i + 1]] = True
    for t, bad in zip((q, k, v, do), (float("nan"), float("inf"), float("nan"), float("-inf"))):
        t[~keep] = bad
    again = _run(q, k, v, do, causal=causal, offsets=offsets)
    for n in want:
        assert torch.equal(again[n][keep], got[n][keep]), n


def _kinds(g, B, N, H, D, device, kinds=5):
    """Queries and keys of a few kinds, so far apart that a query has the same weight for all visible keys of its kind and none for others: the only score that is
    not 0 is 2048, whose product with any scale and whose difference from itself are exact.  Weights are 1 before they are divided, and sums of the values
    exact in fp32.  Values are 64 and something, output gradients 1 and something: delta is a sum of large parts, dS a small difference."""
    kq, kk = (torch.randint(0, kinds, (B, N, H), device=device, generator=g) for _ in range(2))
    kq[:, :kinds] = kk[:, :kinds] = torch.arange(kinds, device=device)[None, :, None]       # (each query sees a key of its kind)
    one = torch.nn.functional.one_hot
    v, do = (c + torch.randn(B, N, H, D, device=device, generator=g) for c in (64, 1))
    return (2048 * one(kq, D)).bfloat16(), one(kk, D).bfloat16(), v.bfloat16(), do.bfloat16()


def _kinds_oracle(q, k, v, do, causal):
    """64-bit outputs and bounds of a sample [N, H, D] of `_kinds`.

    o: sums are exact, the quotient off by 2^-21.  What is kept of o is its rounding and the rounding of the rest, off by B^2 = 2^-16 of o: delta by
    (2^-16 + 2^-21 + D 2^-24) sum |do o|, below 2^-15 of it.  L is some 370 at most and rounded by 2^-16, P by 2^-16 for it and 2^-18 for the exponential
    (a polynomial within 2.7e-6, or two steps of fp32): they are factors of dS.  dS is rounded to bf16."""
    scale, N, e = q.shape[-1] ** -0.5, q.shape[0], 2.0 ** -16 + 2.0 ** -18
    q, k, v, do = (t.double().transpose(0, 1) for t in (q, k, v, do))
    s = q @ k.mT * scale
    if causal:
        s = s.masked_fill(torch.ones(N, N, dtype=torch.bool, device=s.device).triu(1), -math.inf)
    p = torch.softmax(s, -1)
    o = p @ v
    delta, size = ((t * u).sum(-1, keepdim=True) for t, u in ((do, o), (do.abs(), o.abs())))
    ds = p * (do @ v.mT - delta)
    ds_off = (B_STEP + e) * ds.abs() + p * (2.0 ** -15 * size + F_STEP * (do.abs() @ v.abs().mT))
    want = dict(o=o, dq=scale * ds @ k, dk=scale * ds.mT @ q, dv=p.mT @ do)
    off = dict(o=2.0 ** -21 * o.abs(), dq=scale * (ds_off + F_STEP * ds.abs()) @ k.abs(), dk=scale * (ds_off + F_STEP * ds.abs()).mT @ q.abs(),
               dv=((B_STEP + e) * p).mT @ do.abs())
    return {n: t.transpose(0, 1) for n, t in want.items()}, {n: t.transpose(0, 1) for n, t in off.items()}, (p, o, delta)


@pytest.mark.parametrize("N,D", [(300, 64), (384, 96)])
def test_bounds_tell_a_rounded_output_apart(N, D):
    """The gradients of queries with delta from the rounded output alone, or with what the rounding left of the row beside it, are outside the bounds."""
    q, k, v, do = (t[0] for t in _kinds(torch.Generator().manual_seed(3), 1, N, 2, D, "cpu"))
    want, off, (p, o, delta) = _kinds_oracle(q, k, v, do, False)
    d64, k64 = do.double().transpose(0, 1), k.double().transpose(0, 1)
    low = o.bfloat16().double()
    rest = (o - low).bfloat16().double()
    outside = lambda kept: float((((D ** -0.5 * p * (d64 @ v.double().transpose(0, 1).mT - (d64 * kept).sum(-1, keepdim=True))) @ k64).transpose(0, 1)  # noqa: E731
                                  - want["dq"]).abs().gt(off["dq"] + B_STEP * want["dq"].abs()).any(-1).double().mean())
    assert outside(low + rest) == 0
    assert outside(low) > 0.5 and outside(low + rest.roll(1, 1)) > 0.4


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,N,H,D", [(1, 300, 2, 64), (2, 300, 2, 96), (32, 384, 8, 64), (20, 440, 8, 96), (1, 2500, 2, 64), (1, 2500, 1, 96), (1, 1030, 1, 40)])
def test_delta_holds_what_the_output_lost(gen, B, N, H, D, causal):
    """Whole, of one query tile to a CTA, and split over the keys and joined: the gradients need o to 16 bits."""
    q, k, v, do = _kinds(gen, B, N, H, D, "cuda")
    got = _run(q, k, v, do, causal=causal)
    torch.cuda.synchronize()
    _ext.check_device_errors()
    for b in sorted({0, B // 2, B - 1}):
        want, off, _ = _kinds_oracle(q[b], k[b], v[b], do[b], causal)
        for n in want:
            _close(got[n][b], want[n], off[n], f"{n} of sample {b}")


@pytest.mark.gpu
def test_first_call_of_a_process_captured():
    """The device's error word is nobody's graph's: no memory of a graph is left when it and its results are gone, and a replay clears nothing."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    code = """
import torch
from makani_b200.ops import _ext, attention as attn
q = torch.randn(1, 20, 2, 16, device="cuda").bfloat16()
side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.graph(graph, stream=side):
    o = attn.attention(q, q, q)
assert _ext.require().read_error_flag(0) == 0
graph.replay()
torch.cuda.synchronize()
assert torch.equal(o, attn.attention(q, q, q))
_ext.check_device_errors()
del o, graph
torch.cuda.empty_cache()
left = [s for s in torch.cuda.memory_snapshot() if tuple(s["segment_pool_id"]) != (0, 0)]
assert not left, left
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_backward_passes_that_are_refused(gen):
    """Batches of output gradients, and traces of a backward pass, in which the gradients would be constants."""
    from torch.fx.experimental.proxy_tensor import make_fx
    q, k, v, do = _inputs(gen, 2, 20, H=2, Hk=2, D=16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = attn.attention(*leaves)
    with pytest.raises(RuntimeError, match="batches"):
        torch.autograd.grad(o, leaves, torch.stack([do, do]), is_grads_batched=True, retain_graph=True)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda d: torch.autograd.grad(o, leaves, d, retain_graph=True))(do)
    want = torch.autograd.grad(o, leaves, do)
    x = torch.cat([t.flatten(2) for t in leaves], -1).detach().requires_grad_()
    y = attn.attention_qkv(x, 2)
    with pytest.raises(RuntimeError, match="batches"):
        torch.autograd.grad(y, x, torch.stack([do, do]), is_grads_batched=True, retain_graph=True)
    assert torch.equal(torch.autograd.grad(y, x, do)[0], torch.cat([t.flatten(2) for t in want], -1))
