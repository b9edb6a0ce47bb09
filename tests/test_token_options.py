"""The token networks' options together: norms of queries and keys, rotary positions, windows with register tokens, dropout from a counter; as a user of the
recipes has them."""

import pytest
import torch
import torch.nn as nn

from makani_b200.ops import _ext
from makani_b200.ops import attention as attn
from makani_b200.ops import rotary as rot


def _rel(a, b):
    return ((a.double() - b.double()).norm() / (b.double().norm() + 1e-30)).item()


ALL = dict(qk_norm=True, rotary=True, attn_window=2, register_tokens=3)


def _vit(dev, **kw):
    from makani_b200.models.networks.vit import VisionTransformer
    torch.manual_seed(3)
    args = dict(inp_shape=(32, 64), patch_size=(4, 4), inp_chans=5, out_chans=3, embed_dim=96, depth=3, num_heads=4)
    m = VisionTransformer(**{**args, **kw}).to(dev)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.02 * torch.randn_like(p))
    return m


# ---------------------------------------------------------------------------------------------------- any machine

def test_attention_module_with_everything():
    from makani_b200.models.networks.vit import Attention
    torch.manual_seed(1)
    axes, at = rot.RotaryAxes((2, 2), base=50.0), rot.grid_positions(3, 4, first=2)
    m = Attention(24, num_heads=4, qkv_bias=True, qk_norm=True, axes=axes, window=4, sinks=2).eval()
    x = torch.randn(2, 14, 24)
    q, k, v = m.qkv(x).view(2, 14, 3, 4, 6).unbind(2)
    q, k = rot.rotary(m.q_norm(q), at, axes), rot.rotary(m.k_norm(k), at, axes)
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    s = (q @ k.mT / 6 ** 0.5).masked_fill(~attn.visible(14, False, 4, 2), float("-inf"))
    want = m.proj((torch.softmax(s, -1) @ v).transpose(1, 2).reshape(2, 14, 24))
    assert torch.allclose(m(x, at), want, atol=1e-5)
    # a hook on a norm sees it called, with the same outcome
    calls = []
    m.q_norm.register_forward_hook(lambda *a: calls.append(1))
    assert torch.allclose(m(x, at), want, atol=1e-5) and calls
    # dropped weights go through the library, behind the same mask
    m.attn_drop_rate = 1e-9
    assert torch.allclose(m.train()(x, at), want, atol=1e-5)


def test_networks_options_on_the_cpu():
    plain = _vit("cpu")
    assert not {n for n, _ in plain.named_parameters()} & {"registers", "blocks.0.attn.q_norm.weight"} and not list(plain.buffers())
    m = _vit("cpu", **ALL)
    assert m.registers.shape == (1, 3, 96) and m.token_positions.shape == (131, 2) and "token_positions" not in m.state_dict()
    assert m.blocks[0].attn.window == 2 * 16 and m.blocks[0].attn.sinks == 3
    y = m(torch.randn(2, 5, 32, 64))
    assert y.shape == (2, 3, 32, 64)
    y.sum().backward()
    assert all(p.grad is not None for p in m.parameters())
    assert _vit("cpu", attn_window=0)(torch.randn(1, 5, 32, 64)).shape == (1, 3, 32, 64)
    for bad in (-1, 1.5, True):
        with pytest.raises(ValueError, match="attn_window"):
            _vit("cpu", attn_window=bad)
    with pytest.raises(ValueError, match="narrow"):
        _vit("cpu", rotary=True, num_heads=48)
    with pytest.raises(ValueError, match="generators"):
        _vit("cpu", mlp_drop_rate=0.1, dropout_generator="philox")


def test_windows_keep_what_is_far_away():
    """One block sees two rows to either side and the registers: a patch further away does not move."""
    m = _vit("cpu", depth=1, attn_window=2, register_tokens=2).eval()
    x = torch.randn(1, 5, 32, 64)
    y = m(x)
    x[:, :, 28:] += 1.0
    z = m(x)
    assert torch.equal(y[:, :, :16], z[:, :, :16]) and not torch.equal(y[:, :, 20:24], z[:, :, 20:24])


@pytest.mark.parametrize("rows,registers", [(2, 3), (1, 1), (0, 2), (3, 0)])
def test_what_tokens_see_through_a_window(rows, registers):
    """Patches in the first, a middle and the last column, and registers: the farthest row to the north from the own column on, to the south up to it, whole rows in
    between, and all registers; registers see what stands as near to them."""
    m = _vit("cpu", depth=1, attn_window=rows, register_tokens=registers)
    H, W = m.grid
    x = torch.randn(1, registers + H * W, 96, requires_grad=True)
    y = m.blocks[0].attn(x)

    def seen(token):
        g, = torch.autograd.grad(y[0, token].sum(), x, retain_graph=True)
        g = g[0].abs().amax(-1) > 0
        return g[:registers], g[registers:].view(H, W)

    for r in (0, 1, H // 2, H - 1):
        for c in (0, W // 2, W - 1):
            want = torch.zeros(H, W, dtype=torch.bool)
            want[max(r - rows + 1, 0):r + rows] = True
            if r - rows >= 0:
                want[r - rows, c:] = True
            if r + rows < H:
                want[r + rows, :c + 1] = True
            if rows == 0:
                want[:], want[r, c] = False, True
            at, grid = seen(registers + r * W + c)
            assert at.all() and torch.equal(grid, want), (r, c)
    for i in range(registers):
        at, grid = seen(i)
        reach = max(0, i + rows * W - registers + 1)
        assert at.all() and torch.equal(grid.flatten(), torch.arange(H * W) < reach), i


def test_counter_dropout_on_the_cpu():
    m = _vit("cpu", mlp_drop_rate=0.3, dropout_generator="counter")
    x = torch.randn(1, 5, 32, 64)
    assert torch.equal(m.eval()(x), _vit("cpu", mlp_drop_rate=0.3).eval()(x))
    m.train()
    torch.manual_seed(5)
    a = m(x)
    torch.manual_seed(5)
    assert torch.equal(a, m(x)) and not torch.equal(a, m(x))


@pytest.mark.parametrize("where", ["attn", "attn.proj_drop", "drop_path", "mlp", "mlp.fwd", "mlp.fwd.4", "mlp.fwd.3", "all"])
def test_hooks_see_the_calls_of_joint_passes(where):
    """Hooks on what a joint pass takes together: called as often in training as in evaluation, with the module's own result, and the outcome is the same."""
    m = _vit("cpu", depth=1, mlp_drop_rate=0.3, dropout_generator="counter", **ALL)
    x = torch.randn(1, 5, 32, 64)
    torch.manual_seed(5)
    want = m.train()(x)
    seen = []
    hook = lambda mod, args, out: seen.append((args[0].detach(), out.detach()))  # noqa: E731
    if where == "all":
        handle = nn.modules.module.register_module_forward_hook(hook)
    else:
        handle = m.blocks[0].get_submodule(where).register_forward_hook(hook)
    calls = {}
    for training in (True, False):
        seen.clear()
        torch.manual_seed(5)
        y = m.train(training)(x)
        calls[training] = len(seen)
        if training:
            # (watched by all, norms and rotation are calls of their own, each rounded to fp32: some hundred steps of 2^-24 to the end of one block)
            assert torch.equal(y, want) or where == "all" and (y - want).abs().max() < 2.0 ** -16 * want.abs().max()
            if where in ("attn.proj_drop", "mlp.fwd.4"):
                a, b = seen[-1]
                # (dropped, and nothing added; factor and product, and 0.7 and the quotient, are half a step of 2^-24 each)
                assert torch.allclose(b[b != 0], (a / 0.7)[b != 0], rtol=2.0 ** -22, atol=0.0) and 0.1 < (b == 0).double().mean() < 0.5
            if where in ("attn", "mlp", "mlp.fwd"):
                assert 0.1 < (seen[0][1] == 0).double().mean() < 0.5
    handle.remove()
    assert calls[True] == calls[False] > 0
    # with nobody there, the joint pass again
    torch.manual_seed(5)
    assert torch.equal(m.train()(x), want)


def test_joint_passes_are_for_the_classes_that_have_them():
    from makani_b200.models.networks.vit import Attention

    class Mine(Attention):
        def forward(self, x, positions=None):
            return super().forward(x, positions)

    m = _vit("cpu", depth=1, mlp_drop_rate=0.3, dropout_generator="counter")
    x = torch.randn(1, 5, 32, 64)
    torch.manual_seed(5)
    want = m.train()(x)
    m.blocks[0].attn.__class__ = Mine
    torch.manual_seed(5)
    assert torch.equal(m(x), want)


def test_when_forecasts_of_the_mlp_are_fused(monkeypatch):
    """Behind counter dropout: nothing is dropped, nobody watches, and the engine's activation is that of training."""
    from makani_b200.models.common.layers import MLP
    m = MLP(in_features=8, input_format="traditional", drop_rate=0.3, dropout_generator="counter").eval()
    assert m._nothing_dropped() and not m.train()._nothing_dropped() and m.eval()._nothing_dropped()
    handle = m.fwd[1].register_forward_hook(lambda *a: None)
    assert not m._nothing_dropped()
    handle.remove()
    monkeypatch.setattr(_ext, "_GELU_TANH", True)
    assert not m._nothing_dropped()
    assert not MLP(in_features=8, input_format="traditional", drop_rate=0.3).eval()._nothing_dropped()
    monkeypatch.undo()
    for more in (dict(hidden_features=20), dict(out_features=12), dict(act_layer=nn.ReLU)):
        assert not MLP(in_features=8, input_format="traditional", drop_rate=0.3, dropout_generator="counter", **more).eval()._nothing_dropped()


@pytest.mark.parametrize("name", ["vit_73chq_window"])
def test_recipe(name):
    from makani_b200.utils.YParams import YParams
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = YParams(os.path.join(root, "config", "vit.yaml"), name)
    assert p.qk_norm and p.rotary and p.attn_window > 0 and p.register_tokens > 0 and p.dropout_generator == "counter"


# ---------------------------------------------------------------------------------------------------- the kernels

@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.available()
    yield torch.device("cuda", 0)
    torch.cuda.synchronize()
    _ext.check_device_errors()


def _pass(m, x, dy, autocast, native):
    _ext.set_native(native)
    try:
        m.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y = m(x)
        y.backward(dy.to(y.dtype))
        return y.detach().float(), {n: p.grad.detach().float().clone() for n, p in m.named_parameters()}
    finally:
        _ext.set_native(True)


OPTIONS = [dict(qk_norm=True, rotary=True), dict(rotary=True, attn_window=2), dict(attn_window=1, register_tokens=4), ALL,
           dict(ALL, embed_dim=256, num_heads=2, inp_shape=(64, 128))]


@pytest.mark.gpu
@pytest.mark.parametrize("options", OPTIONS)
def test_networks_against_fp32(dev, options):
    """Under autocast, the native pass is no further from the fp32 formulation than torch's own bf16 pass is, give or take a half."""
    m = _vit(dev, **options)
    g = torch.Generator(dev).manual_seed(5)
    H, W = options.get("inp_shape", (32, 64))
    x = torch.randn(2, 5, H, W, device=dev, generator=g)
    dy = torch.randn(2, 3, H, W, device=dev, generator=g)
    y0, g0 = _pass(m, x, dy, False, False)
    y1, g1 = _pass(m, x, dy, True, False)
    before = _ext.launch_count()
    y2, g2 = _pass(m, x, dy, True, True)
    assert _ext.launch_count() > before
    assert _rel(y2, y0) < 1.5 * _rel(y1, y0) + 1e-3
    for n in g0:
        assert _rel(g2[n], g0[n]) < 1.5 * _rel(g1[n], g0[n]) + 1e-2, n


@pytest.mark.gpu
def test_no_library_attention_norm_or_dropout(dev, monkeypatch):
    m = _vit(dev, **ALL, mlp_drop_rate=0.1, dropout_generator="counter")

    def refuse(*a, **k):
        raise AssertionError("library call")

    for name in ("scaled_dot_product_attention", "layer_norm", "dropout"):
        monkeypatch.setattr(torch.nn.functional, name, refuse)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(torch.randn(1, 5, 32, 64, device=dev))
    y.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("training", [True, False])
def test_no_library_products_behind_counter_dropout(dev, training, monkeypatch):
    """Both layers of the MLP on the engine, too, in training and in forecasts; and its forecast is that of the network without dropout."""
    m = _vit(dev, **ALL, mlp_drop_rate=0.1, dropout_generator="counter").train(training)
    x = torch.randn(1, 5, 32, 64, device=dev)

    def refuse(*a, **k):
        raise AssertionError("library call")

    with torch.autocast("cuda", dtype=torch.bfloat16):
        if not training:
            want = _vit(dev, **ALL).eval()(x)
        for name in ("linear", "scaled_dot_product_attention", "layer_norm", "dropout"):
            monkeypatch.setattr(torch.nn.functional, name, refuse)
        y = m(x)
    assert training or torch.equal(y, want)
    y.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("joint", [True, False])
def test_mlp_behind_counter_dropout(dev, joint):
    """Values and gradients of the MLP in training against the formula in 64 bits, with the masks that the generator draws: each product, activation and sum is
    rounded to bf16, 2^-9 of the size on average, four of them one behind the other and as many in the backward pass: 2^-7 in all."""
    from makani_b200.models.common.layers import MLP
    torch.manual_seed(2)
    m = MLP(in_features=64, hidden_features=256, input_format="traditional", drop_rate=0.3, dropout_generator="counter").to(dev)
    x, r = (torch.randn(2, 300, 64, device=dev).bfloat16().requires_grad_() for _ in range(2))
    dy = torch.randn(2, 300, 64, device=dev).bfloat16()
    torch.manual_seed(9)
    keep = [m.fwd[2](torch.ones(2, 300, c, device=dev)).double() for c in (256, 64)]
    torch.manual_seed(9)
    y = m(x, r) if joint else m(x)
    grads = torch.autograd.grad(y, [x, *m.parameters()], dy)
    x64, p64 = x.detach().double().requires_grad_(), [p.detach().double().requires_grad_() for p in m.parameters()]
    h = torch.nn.functional.gelu(x64 @ p64[0].bfloat16().double().T + p64[1])
    want = (h * keep[0] @ p64[2].bfloat16().double().T + p64[3]) * keep[1] + (r.detach().double() if joint else 0.0)
    assert _rel(y.detach(), want.detach()) < 2.0 ** -7
    for got, ref in zip(grads, torch.autograd.grad(want, [x64, *p64], dy.double())):
        assert _rel(got, ref) < 2.0 ** -7
    # dropouts alone in training, as for several draws of one forecast, still drop
    m.eval()
    plain = m(x)
    m.fwd[2].train()
    assert not torch.equal(m(x), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,out", [(20, 16), (24, 12), (24, 16)])
def test_widths_of_the_mlp_behind_counter_dropout(dev, hidden, out):
    """Widths that are no multiple of eight, in training and in forecasts."""
    from makani_b200.models.common.layers import MLP
    torch.manual_seed(2)
    m = MLP(in_features=16, hidden_features=hidden, out_features=out, input_format="traditional", drop_rate=0.3, dropout_generator="counter").to(dev).eval()
    x = torch.randn(2, 50, 16, device=dev).bfloat16().requires_grad_()
    p = [t.detach().double() for t in m.parameters()]
    want = torch.nn.functional.gelu(x.detach().double() @ p[0].bfloat16().double().T + p[1]) @ p[2].bfloat16().double().T + p[3]
    assert _rel(m(x).detach(), want) < 2.0 ** -7
    m.train()(x).float().sum().backward()
    assert all(torch.isfinite(t.grad).all() for t in (x, *m.parameters()))


@pytest.mark.gpu
def test_counter_dropout_has_one_mask_both_ways(dev):
    """In fp32, a step along the gradient changes the output by what the gradient says, with the masks of one seed."""
    m = _vit(dev, mlp_drop_rate=0.2, dropout_generator="counter", **ALL).train()
    g = torch.Generator(dev).manual_seed(5)
    x, dy = torch.randn(1, 5, 32, 64, device=dev, generator=g), torch.randn(1, 3, 32, 64, device=dev, generator=g)

    def loss():
        torch.manual_seed(8)
        return (m(x).double() * dy.double()).sum()

    value = loss()
    value.backward()
    assert torch.equal(value, loss())
    grads = {n: p.grad.clone() for n, p in m.named_parameters()}
    norm = sum(v.double().square().sum() for v in grads.values()).sqrt().item()
    h, moved = 1e-2, []
    for sign in (1, -1):
        with torch.no_grad():
            for n, p in m.named_parameters():
                p.add_(sign * h / norm * grads[n])
            moved.append(loss().item())
            for n, p in m.named_parameters():
                p.sub_(sign * h / norm * grads[n])
    # (the third derivative leaves h^2 of the slope, fp32 some 1e-6 of the sum of 6144 terms over the difference)
    assert abs((moved[0] - moved[1]) / (2 * h) - norm) < 2e-2 * norm


@pytest.mark.gpu
def test_captured_step_with_everything(dev):
    """A training step in a CUDA graph: replays go on learning, with new masks each time, and the loss stays finite."""
    m = _vit(dev, mlp_drop_rate=0.1, dropout_generator="counter", **ALL).train()
    opt = torch.optim.SGD(m.parameters(), lr=1e-3)
    x, t = torch.randn(1, 5, 32, 64, device=dev), torch.randn(1, 3, 32, 64, device=dev)

    def step():
        opt.zero_grad(set_to_none=False)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = (m(x).float() - t).square().mean()
        loss.backward()
        opt.step()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = step()
    torch.cuda.current_stream().wait_stream(side)
    before = [p.detach().clone() for p in m.parameters()]
    seen = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(loss.item())
    assert all(torch.isfinite(torch.tensor(v)) for v in seen) and len(set(seen)) == 4
    assert all(not torch.equal(a, p) for a, p in zip(before, m.parameters()))


def _compiled_calls(dev):
    """Every operator with a node of its own: (call, leaves)."""
    from makani_b200.ops import dropout as drop
    g = torch.Generator(dev).manual_seed(5)
    leaf = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device=dev, generator=g).to(dtype).requires_grad_()  # noqa: E731
    axes, at = rot.RotaryAxes((8, 4)), torch.rand(60, 2, device=dev, generator=g)
    q, k, v, qkv = leaf(1, 60, 4, 16), leaf(1, 60, 2, 16), leaf(1, 60, 2, 16), leaf(1, 60, 8 * 16)
    flat = qkv.detach()[0].requires_grad_()
    off = torch.tensor([0, 13, 13, 55], dtype=torch.int32, device=dev)
    p = [leaf(16, dtype=torch.float32) for _ in range(4)]
    x, r, seed = leaf(50, 40), leaf(50, 40, dtype=torch.float32), torch.tensor([3, 4], device=dev)
    return {
        "attention": (lambda: attn.attention(q, k, v), [q, k, v]),
        "window": (lambda: attn.attention(q, k, v, causal=True, window=7, sinks=2), [q, k, v]),
        "projection": (lambda: attn.attention_qkv(flat, 4, 2, offsets=off, window=(9, 3), scale=0.3), [flat]),
        "rotation": (lambda: rot.rotary_qk(q, k, at, axes), [q, k]),
        "rotation back": (lambda: rot.rotary(q, at, axes, inverse=True), [q]),
        "norms": (lambda: rot.norm_rotary_qk(q, k, p[0], p[1], at, axes, p[2], p[3], eps=1e-3, norm="rms"), [q, k, *p]),
        "norms without weights": (lambda: rot.norm_rotary_qk(q, k, None, None), [q, k]),
        "path": (lambda: rot.rotary_attention_qkv(qkv, 4, 2, at, axes, window=7, sinks=1), [qkv]),
        "path with norms": (lambda: rot.rotary_attention_qkv(flat, 4, 2, at, axes, *p, norm="layer", offsets=off, window=7, sinks=1), [flat, *p]),
        "dropout": (lambda: drop.dropout(x, 0.3, seed=seed), [x]),
        "dropout of the generator": (lambda: drop.dropout(x, 0.3), [x]),
        "dropout and sum": (lambda: drop.dropout_add(x, r, 0.3, seed=seed), [x, r]),
        "sum in bf16": (lambda: drop.dropout_add(r, x, 0.3, seed=seed), [x, r]),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attention", "window", "projection", "rotation", "rotation back", "norms", "norms without weights", "path", "path with norms", "dropout",
                                  "dropout of the generator", "dropout and sum", "sum in bf16"])
def test_compiled_backward_passes(dev, name):
    """A backward pass that is compiled calls the kernels with what the node keeps: the same bits, again with other tensors of the same sizes."""
    from torch._dynamo import compiled_autograd
    call, leaves = _compiled_calls(dev)[name]

    def grads():
        torch.manual_seed(6)
        out = call()
        out = (out,) if isinstance(out, torch.Tensor) else tuple(out)
        return torch.autograd.grad(sum(t.float().square().sum() for t in out), leaves)

    for _ in range(2):
        before = _ext.launch_count()
        want = grads()
        launches = _ext.launch_count() - before
        with compiled_autograd._enable(torch.compile(backend="eager")):
            got = grads()
        assert _ext.launch_count() - before == 2 * launches > 0
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        with torch.no_grad():
            for t in leaves:
                t.add_(torch.randn_like(t))
