"""Building blocks shared by the networks: stochastic depth, patch embedding, pointwise encoder/decoder and
MLP stacks, and the planar FFT wrappers used by the FNO variants.

Module and parameter names follow the reference (makani/models/common/layers.py:35-287) so that its
checkpoints load: `EncoderDecoder.fwd.{0,2}`, `MLP.fwd.{0,3}`.  On CUDA bf16 inputs the two-layer stacks run
as fused tcgen05 GEMM chains (`makani_b200.ops.conv.mlp2`); otherwise as plain torch modules.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

from ...ops import _ext
from ...ops import conv as conv_ops
from ...ops import dropout as dropout_ops
from ...ops import linear as linear_ops


def drop_path(x: torch.Tensor, drop_prob: float = 0.0, training: bool = False) -> torch.Tensor:
    """Per-sample stochastic depth."""
    if drop_prob == 0.0 or not training:
        return x
    keep = 1.0 - drop_prob
    shape = (x.shape[0],) + (1,) * (x.ndim - 1)
    mask = keep + torch.rand(shape, dtype=x.dtype, device=x.device)
    mask.floor_()
    return x.div(keep) * mask


class DropPath(nn.Module):
    def __init__(self, drop_prob=None):
        super().__init__()
        self.drop_prob = drop_prob

    def forward(self, x):
        return drop_path(x, self.drop_prob, self.training)


def watched(m: nn.Module, forward) -> bool:
    """Whether somebody has to see the call of a module: hooks, its own or of all modules, or another class's `forward`, for which joint passes stay apart."""
    g = nn.modules.module
    return bool(m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks or g._global_forward_hooks or g._global_forward_pre_hooks
                or g._global_backward_hooks or g._global_backward_pre_hooks or "forward" in m.__dict__ or type(m).forward is not forward)


class Dropout(nn.Dropout):
    """`nn.Dropout` on the kernel of `ops/dropout.py`, whose mask is made again in the backward pass instead of being kept (and is another than torch's)."""

    def __init__(self, p: float = 0.5):
        super().__init__(p)

    def forward(self, x):
        return dropout_ops.dropout(x, self.p, self.training)

    def add(self, x, residual):
        """residual + dropout(x), in one pass over memory."""
        return dropout_ops.dropout_add(x, residual, self.p, self.training)

    def joins(self) -> bool:
        """Whether `add` may take its place: it drops something, and nobody has to see its call."""
        return self.training and not watched(self, Dropout.forward)


def dropout_layer(p: float, generator: str = "torch") -> nn.Module:
    """`generator` "torch": torch's dropout; "counter": the one above."""
    if generator not in ("torch", "counter"):
        raise ValueError(f"dropout generators are torch and counter, got {generator!r}")
    if p <= 0.0:
        return nn.Identity()
    return Dropout(p) if generator == "counter" else nn.Dropout(p)


class PatchEmbed(nn.Module):
    def __init__(self, img_size=(224, 224), patch_size=(16, 16), in_chans=3, embed_dim=768):
        super().__init__()
        self.img_size = img_size
        self.patch_size = patch_size
        self.red_img_size = (img_size[0] // patch_size[0], img_size[1] // patch_size[1])
        self.num_patches = self.red_img_size[0] * self.red_img_size[1]
        self.proj = nn.Conv2d(in_chans, embed_dim, kernel_size=patch_size, stride=patch_size)
        self.proj.weight.is_shared_mp = ["spatial"]
        self.proj.bias.is_shared_mp = ["spatial"]

    def forward(self, x):
        B, C, H, W = x.shape
        assert H == self.img_size[0] and W == self.img_size[1], f"Input image size ({H}*{W}) doesn't match model ({self.img_size[0]}*{self.img_size[1]})."
        # [B, C, H, W] -> [B, embed, H/p * W/p]
        return self.proj(x).flatten(2)


def _is_gelu(act_layer) -> bool:
    return act_layer is nn.GELU


class EncoderDecoder(nn.Module):
    """`num_layers` x (pointwise linear + bias + activation) followed by a bias-free pointwise linear."""

    def __init__(self, num_layers, input_dim, output_dim, hidden_dim, act_layer, gain=1.0, input_format="nchw"):
        super().__init__()
        mods = []
        cur = input_dim
        for _ in range(num_layers):
            lin = nn.Conv2d(cur, hidden_dim, 1, bias=True) if input_format == "nchw" else nn.Linear(cur, hidden_dim, bias=True)
            nn.init.normal_(lin.weight, mean=0.0, std=math.sqrt(2.0 / cur))
            nn.init.constant_(lin.bias, 0.0)
            lin.weight.is_shared_mp = ["spatial"]
            lin.bias.is_shared_mp = ["spatial"]
            mods += [lin, act_layer()]
            cur = hidden_dim
        out = nn.Conv2d(cur, output_dim, 1, bias=False) if input_format == "nchw" else nn.Linear(cur, output_dim, bias=False)
        nn.init.normal_(out.weight, mean=0.0, std=math.sqrt(gain / cur))
        out.weight.is_shared_mp = ["spatial"]
        mods.append(out)
        self.fwd = nn.Sequential(*mods)
        self._fusable = (num_layers == 1 and input_format == "nchw" and _is_gelu(act_layer))

    def forward(self, x):
        if self._fusable and x.is_cuda and conv_ops.fast_path_ok(x):
            return conv_ops.mlp2(x, self.fwd[0].weight, self.fwd[0].bias, self.fwd[2].weight, None)
        return self.fwd(x)


class TokenLinear(nn.Linear):
    """`nn.Linear` whose product runs on the GEMM engine where the tokens qualify (`ops/linear.py`)."""

    def forward(self, x):
        return linear_ops.linear_lastdim(x, self.weight, self.bias)


class MLP(nn.Module):
    """fc1 -> act -> drop -> fc2 -> drop, pointwise over NCHW (1x1 convs) or the last dim ("traditional")."""

    def __init__(self, in_features, hidden_features=None, out_features=None, act_layer=nn.GELU, output_bias=True,
                 input_format="nchw", drop_rate=0.0, drop_type="iid", checkpointing=0, gain=1.0, dropout_generator="torch", **kwargs):
        super().__init__()
        self.checkpointing = checkpointing
        out_features = out_features or in_features
        hidden_features = hidden_features or in_features
        counter = drop_rate > 0.0 and dropout_generator == "counter" and drop_type == "iid" and input_format == "traditional"
        if input_format == "nchw":
            fc1 = nn.Conv2d(in_features, hidden_features, 1, bias=True)
            fc2 = nn.Conv2d(hidden_features, out_features, 1, bias=output_bias)
            for p in list(fc1.parameters()) + list(fc2.parameters()):
                p.is_shared_mp = ["spatial"]
        elif input_format == "traditional":
            if drop_type == "features":
                raise NotImplementedError("feature dropout needs the nchw format")
            # (behind torch's own dropout torch's own products)
            linear = TokenLinear if counter else nn.Linear
            fc1 = linear(in_features, hidden_features, bias=True)
            fc2 = linear(hidden_features, out_features, bias=output_bias)
        else:
            raise NotImplementedError(f"input format {input_format} not supported")
        nn.init.normal_(fc1.weight, mean=0.0, std=math.sqrt(2.0 / in_features))
        nn.init.constant_(fc1.bias, 0.0)
        nn.init.normal_(fc2.weight, mean=0.0, std=math.sqrt(gain / hidden_features))
        if fc2.bias is not None:
            nn.init.constant_(fc2.bias, 0.0)
        if drop_rate > 0.0:
            drop = dropout_layer(drop_rate, dropout_generator) if drop_type == "iid" else nn.Dropout2d(drop_rate)
        else:
            drop = nn.Identity()
        self.fwd = nn.Sequential(fc1, act_layer(), drop, fc2, drop)
        self._fusable = (input_format == "nchw" and _is_gelu(act_layer) and drop_rate == 0.0)
        self._fusable_tokens = (input_format == "traditional" and _is_gelu(act_layer) and drop_rate == 0.0)
        self._fusable_forecasts = counter and _is_gelu(act_layer) and hidden_features % 8 == 0 and out_features % 8 == 0

    def _run(self, x):
        if self._fusable and x.is_cuda and conv_ops.fast_path_ok(x):
            return conv_ops.mlp2(x, self.fwd[0].weight, self.fwd[0].bias, self.fwd[3].weight, self.fwd[3].bias)
        if (self._fusable_tokens or self._nothing_dropped()) and linear_ops.fast_path_ok(x):
            return linear_ops.mlp2_lastdim(x, self.fwd[0].weight, self.fwd[0].bias, self.fwd[3].weight, self.fwd[3].bias)
        return self.fwd(x)

    def _nothing_dropped(self) -> bool:
        """Whether the dropouts leave everything as it is, and nobody has to see them, or the layers around them, called."""
        # (the activation as in training: the engine's other form is for networks that have it throughout)
        return self._fusable_forecasts and not self.fwd[2].training and _ext.gelu_approximation() == "none" and not any(watched(m, type(m).forward) for m in (self.fwd, *self.fwd))

    def checkpoint_forward(self, x):
        """The forward pass with its activations recomputed in backward (makani/models/common/layers.py `MLP`)."""
        return checkpoint(self._run, x, use_reentrant=False)

    def forward(self, x, residual=None):
        """The stack of x; with a residual, their sum, which takes the last dropout with it where that can."""
        if self.checkpointing >= 2 and self.training:
            y = self.checkpoint_forward(x)
        elif residual is not None and isinstance(self.fwd[4], Dropout) and self.fwd[4].joins() and not watched(self.fwd, nn.Sequential.forward):
            for i in range(4):
                x = self.fwd[i](x)
            return self.fwd[4].add(x, residual)
        else:
            y = self._run(x)
        return y if residual is None else residual + y


class RealFFT2(nn.Module):
    """rfft2 (ortho) truncated to the `lmax` lowest |k_lat| rows and first `mmax` columns."""

    def __init__(self, nlat, nlon, lmax=None, mmax=None):
        super().__init__()
        self.nlat, self.nlon = nlat, nlon
        self.lmax = min(lmax or nlat, nlat)
        self.mmax = min(mmax or nlon // 2 + 1, nlon // 2 + 1)
        self.truncate = not (self.lmax == nlat and self.mmax == nlon // 2 + 1)
        self.lmax_high = math.ceil(self.lmax / 2)
        self.lmax_low = math.floor(self.lmax / 2)

    def forward(self, x):
        y = torch.fft.rfft2(x, s=(self.nlat, self.nlon), dim=(-2, -1), norm="ortho")
        if self.truncate:
            parts = [y[..., : self.lmax_high, : self.mmax]]
            if self.lmax_low > 0:
                parts.append(y[..., -self.lmax_low:, : self.mmax])
            y = torch.cat(parts, dim=-2)
        return y


class InverseRealFFT2(nn.Module):
    """Inverse of `RealFFT2`: zero-pads the discarded middle rows, then irfft2 (ortho)."""

    def __init__(self, nlat, nlon, lmax=None, mmax=None):
        super().__init__()
        self.nlat, self.nlon = nlat, nlon
        self.lmax = min(lmax or nlat, nlat)
        self.mmax = min(mmax or nlon // 2 + 1, nlon // 2 + 1)
        self.truncate = not (self.lmax == nlat and self.mmax == nlon // 2 + 1)
        self.lmax_high = math.ceil(self.lmax / 2)
        self.lmax_low = math.floor(self.lmax / 2)

    def forward(self, x):
        xt = x[..., : self.mmax]
        if self.truncate:
            hi = F.pad(xt[..., : self.lmax_high, :], (0, 0, 0, self.nlat - self.lmax))
            parts = [hi]
            if self.lmax_low > 0:
                parts.append(xt[..., -self.lmax_low:, :])
            xt = torch.cat(parts, dim=-2)
        return torch.fft.irfft2(xt, s=(self.nlat, self.nlon), dim=(-2, -1), norm="ortho")
