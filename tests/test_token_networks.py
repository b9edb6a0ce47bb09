"""Layer norm and attention as the token networks use them together: ViT and AFNO against their plain torch formulation, the norms' modules, and
a captured training step."""

import pytest
import torch
import torch.nn as nn

from makani_b200.ops import _ext


def _rel(a, b):
    return ((a.double() - b.double()).norm() / (b.double().norm() + 1e-30)).item()


# ---------------------------------------------------------------------------------------------------- any machine

def test_layer_norm_module_is_torchs():
    from makani_b200.parallel.layer_norm import LayerNorm, normed
    torch.manual_seed(0)
    ours, theirs = LayerNorm(12, eps=1e-6), nn.LayerNorm(12, eps=1e-6)
    with torch.no_grad():
        for p in theirs.parameters():
            p.normal_()
    ours.load_state_dict(theirs.state_dict())
    x, r = torch.randn(3, 5, 12), torch.randn(3, 5, 12)
    assert torch.equal(ours(x), theirs(x))
    s, y = ours.after_sum(x, r)
    assert torch.equal(s, x + r) and torch.equal(y, theirs(x + r))
    assert normed(ours, x, torch.bfloat16).dtype == normed(theirs, x, torch.bfloat16).dtype == torch.bfloat16
    with pytest.raises(ValueError, match="12 channels"):
        ours(torch.randn(3, 1))
    with pytest.raises(ValueError, match="12 channels"):
        ours.after_sum(torch.randn(3, 1), torch.randn(3, 1))
    two = LayerNorm((5, 12))
    assert torch.equal(two(x), nn.LayerNorm((5, 12))(x)) and torch.equal(two.after_sum(x, r)[1], two(x + r))


@pytest.mark.parametrize("qk_norm", [False, True])
def test_attention_module_on_cpu(qk_norm):
    from makani_b200.models.networks.vit import Attention
    torch.manual_seed(1)
    m = Attention(24, num_heads=4, qkv_bias=True, qk_norm=qk_norm).eval()
    x = torch.randn(2, 9, 24)
    q, k, v = m.qkv(x).view(2, 9, 3, 4, 6).permute(2, 0, 3, 1, 4).unbind(0)
    want = torch.softmax(m.q_norm(q) @ m.k_norm(k).mT / 6 ** 0.5, -1) @ v
    assert torch.allclose(m(x), m.proj(want.transpose(1, 2).reshape(2, 9, 24)), atol=1e-5)


# ---------------------------------------------------------------------------------------------------- the kernels

@pytest.fixture
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    assert _ext.available()
    return torch.device("cuda", 0)


def _vit(dev, **kw):
    from makani_b200.models.networks.vit import VisionTransformer
    torch.manual_seed(3)
    args = dict(inp_shape=(32, 64), patch_size=(4, 4), inp_chans=5, out_chans=3, embed_dim=96, depth=3, num_heads=4)
    m = VisionTransformer(**{**args, **kw}).to(dev)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.02 * torch.randn_like(p))
    return m


def _afno(dev, **kw):
    from makani_b200.models.networks.afnonet import AdaptiveFourierNeuralOperatorNet as AFNO
    torch.manual_seed(4)
    m = AFNO(inp_shape=(32, 64), patch_size=(4, 4), inp_chans=5, out_chans=3, embed_dim=64, num_layers=2, num_blocks=4, **kw).to(dev)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.02 * torch.randn_like(p))
    return m


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


@pytest.mark.gpu
@pytest.mark.parametrize("make", [_vit, _afno])
def test_networks_against_fp32(dev, make):
    """Under autocast, the native pass is no further from the fp32 formulation than torch's own bf16 pass is, give or take a half."""
    m = make(dev)
    g = torch.Generator(dev).manual_seed(5)
    x = torch.randn(2, 5, 32, 64, device=dev, generator=g)
    dy = torch.randn(2, 3, 32, 64, device=dev, generator=g)
    y0, g0 = _pass(m, x, dy, False, False)
    y1, g1 = _pass(m, x, dy, True, False)
    before = _ext.launch_count()
    y2, g2 = _pass(m, x, dy, True, True)
    assert _ext.launch_count() > before
    torch.cuda.synchronize()
    _ext.check_device_errors(dev)
    assert _rel(y2, y0) < 1.5 * _rel(y1, y0) + 1e-3
    for n in g0:
        assert _rel(g2[n], g0[n]) < 1.5 * _rel(g1[n], g0[n]) + 1e-2, n


@pytest.mark.gpu
def test_vit_calls_no_library_attention_or_norm(dev, monkeypatch):
    m = _vit(dev)

    def refuse(*a, **k):
        raise AssertionError("library call")

    monkeypatch.setattr(torch.nn.functional, "scaled_dot_product_attention", refuse)
    monkeypatch.setattr(torch.nn.functional, "layer_norm", refuse)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        m(torch.randn(1, 5, 32, 64, device=dev)).float().sum().backward()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_vit_in_fp32_and_with_dropout_keeps_to_torch(dev):
    """Without autocast nothing of the network changes but the norms' sums; attention dropout in training stays the library's."""
    m = _vit(dev)
    x = torch.randn(2, 5, 32, 64, device=dev)
    y0, g0 = _pass(m, x, torch.ones(2, 3, 32, 64, device=dev), False, False)
    y1, g1 = _pass(m, x, torch.ones(2, 3, 32, 64, device=dev), False, True)
    assert _rel(y1, y0) < 1e-5 and all(_rel(g1[n], g0[n]) < 1e-3 for n in g0)
    d = _vit(dev, attn_drop_rate=0.5).train()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert not torch.equal(d(x), d(x))
        d.eval()
        assert torch.equal(d(x), d(x))


@pytest.mark.gpu
def test_query_and_key_norms(dev):
    """Norms of strided heads between projection and attention, with every gradient."""
    from makani_b200.models.networks.vit import Attention
    torch.manual_seed(6)
    m = Attention(96, num_heads=4, qkv_bias=True, qk_norm=True).to(dev)
    x = torch.randn(2, 150, 96, device=dev)
    dy = torch.randn(2, 150, 96, device=dev)
    y0, g0 = _pass(m, x, dy, False, False)
    y1, g1 = _pass(m, x, dy, True, False)
    y2, g2 = _pass(m, x.bfloat16(), dy, True, True)
    assert _rel(y2, y0) < 1.5 * _rel(y1, y0) + 1e-3
    for n in g0:
        assert _rel(g2[n], g0[n]) < 1.5 * _rel(g1[n], g0[n]) + 1e-2, n


@pytest.mark.gpu
@pytest.mark.parametrize("channels_last", [False, True])
def test_distributed_layer_norm_on_one_rank(dev, channels_last):
    from makani_b200.parallel.layer_norm import DistributedLayerNorm
    torch.manual_seed(7)
    m = DistributedLayerNorm(40, eps=1e-6).to(dev)
    with torch.no_grad():
        for p in m.parameters():
            p.normal_()
    x = torch.randn(2, 40, 9, 14, device=dev).bfloat16()
    x = (x.contiguous(memory_format=torch.channels_last) if channels_last else x).requires_grad_()
    y = m(x)
    want = torch.nn.functional.layer_norm(x.detach().double().permute(0, 2, 3, 1), (40,), m.norm.weight.double(), m.norm.bias.double(), 1e-6)
    assert y.dtype == torch.bfloat16 and _rel(y, want.permute(0, 3, 1, 2)) < 2.0 ** -8
    y.sum().backward()
    assert x.grad.shape == x.shape
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert m(x).dtype == torch.float32


@pytest.mark.gpu
def test_captured_step_follows_eager_steps(dev):
    """Forward, backward and AdamW of a ViT replayed from one graph, against eager launches."""
    from makani_b200.ops.optim import FusedAdamW
    from makani_b200.parallel.grad_reduce import GradReducer
    from makani_b200.utils.train_step import GraphedTrainStep, TrainStep

    class Autocast(nn.Module):
        def __init__(self, net):
            super().__init__()
            self.net = net

        def forward(self, x):
            with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
                return self.net(x)

    def run(cls):
        m = Autocast(_vit(dev, depth=2))
        red = GradReducer(m)
        opt = FusedAdamW(m.parameters(), lr=1e-3)
        step = cls(m, lambda p, t, i: (p.float() - t.float()).square().mean(), opt, red)
        g = torch.Generator(device=dev).manual_seed(9)
        losses = []
        for _ in range(6):
            losses.append(float(step(torch.randn(2, 5, 32, 64, device=dev, generator=g), torch.randn(2, 3, 32, 64, device=dev, generator=g))))
        torch.cuda.synchronize()
        return losses, step

    eager, _ = run(TrainStep)
    replayed, step = run(GraphedTrainStep)
    assert step.graph is not None
    _ext.check_device_errors(dev)
    for a, b in zip(eager, replayed):
        assert abs(a - b) < 2e-2 * max(1.0, abs(a)), (eager, replayed)


@pytest.mark.parametrize("make", [_vit, _afno])
def test_hooks_of_every_norm_are_called(make):
    """Hooks see the calls of a plain module, one tensor in and one out, and may change either; what they see is what the network computes with."""
    m = make("cpu")
    x = torch.randn(1, 5, 32, 64)
    want = m(x)
    norms = {n: mod for n, mod in m.named_modules() if isinstance(mod, nn.LayerNorm)}
    assert any("norm2" in n for n in norms)
    calls = {n: [] for n in norms}
    handles = []
    for n, mod in norms.items():
        handles.append(mod.register_forward_pre_hook(lambda mod, args, n=n: calls[n].append(("pre", len(args), args[0].shape))))
        handles.append(mod.register_forward_hook(lambda mod, args, y, n=n: calls[n].append(("post", len(args), y.shape))))
        handles.append(mod.register_full_backward_hook(lambda mod, gi, go, n=n: calls[n].append(("back", len(go), go[0].shape))))
    y = m(x)
    assert torch.equal(y, want)
    y.sum().backward()
    for n, seen in calls.items():
        assert [(kind, count) for kind, count, _ in seen] == [("pre", 1), ("post", 1), ("back", 1)], (n, seen)
        assert len({shape for _, _, shape in seen}) == 1
    for h in handles:
        h.remove()
    second = [mod for n, mod in norms.items() if "norm2" in n]
    handles = [mod.register_forward_hook(lambda mod, args, y: 2 * y) for mod in second]
    with torch.no_grad():
        doubled = m(x)
        for h in handles:
            h.remove()
        for mod in second:
            mod.weight.mul_(2)
            mod.bias.mul_(2)
        assert not torch.equal(doubled, want) and torch.equal(doubled, m(x))


def test_a_norm_with_a_forward_of_its_own():
    from makani_b200.parallel.layer_norm import LayerNorm, normed

    class Shifted(LayerNorm):
        def forward(self, x, out_dtype=None):
            return super().forward(x, out_dtype) + 1

    torch.manual_seed(0)
    m = Shifted(12)
    x, r = torch.randn(3, 12), torch.randn(3, 12)
    s, y = m.after_sum(x, r)
    assert torch.equal(s, x + r) and torch.equal(y, m(x + r))
    plain = LayerNorm(12)
    plain.forward = lambda x, out_dtype=None: x * 3
    assert torch.equal(plain.after_sum(x, r)[1], (x + r) * 3) and torch.equal(normed(plain, x, torch.float32), x * 3)


def test_sums_in_the_wider_type_stay_there():
    """`after_sum` of two types hands on what the sum's type is, whichever of the two has it."""
    from makani_b200.parallel.layer_norm import LayerNorm
    m = LayerNorm(12)
    for a, b in ((torch.float64, torch.float32), (torch.float32, torch.float64), (torch.float64, torch.bfloat16), (torch.bfloat16, torch.float32),
                 (torch.float32, torch.float16), (torch.float16, torch.bfloat16)):
        wide = torch.promote_types(a, b)
        s, y = m.after_sum(torch.randn(3, 12).to(a), torch.randn(3, 12).to(b))
        assert s.dtype == y.dtype == wide, (a, b, s.dtype, y.dtype)


def test_networks_without_memory():
    """Shapes and types on the meta device, as torch's own modules give them."""
    from makani_b200.parallel.layer_norm import LayerNorm
    m = LayerNorm(12).to("meta")
    s, y = m.after_sum(torch.randn(3, 12, device="meta"), torch.randn(3, 12, device="meta"))
    assert s.shape == y.shape == (3, 12) and y.is_meta
    y = _vit("cpu").to("meta")(torch.randn(2, 5, 32, 64, device="meta"))
    assert y.is_meta and y.shape == (2, 3, 32, 64)


def test_norm_under_autocast_of_the_cpu():
    """As torch's norm there: the types are those of the call."""
    from makani_b200.parallel.layer_norm import LayerNorm
    ours, theirs = LayerNorm(12), nn.LayerNorm(12)
    x = torch.randn(3, 12)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert ours(x).dtype == theirs(x).dtype and torch.equal(ours(x), theirs(x))
        assert ours(x, torch.bfloat16).dtype == torch.bfloat16
