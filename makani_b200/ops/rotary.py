"""Rotary positions with several axes (time, height, width, ...) for queries and keys, alone or behind a norm of every head's channels, in one pass
over memory in either direction; and a fused projection's way through both into attention.

Layout as in `ops/attention.py`: tokens first, heads inside, [B, N, heads, D] or packed [T, heads, D].  The channels of a head are split into bands, one per
axis, one after the other from the first channel on; pair i of a band of b channels turns by the angle position[axis] * base^(-2 i / b).  Channels behind
the bands stay as they are.  Pairs are the halves of a band (i, i + b / 2), or, interleaved, neighbours (2 i, 2 i + 1).

Positions are whole numbers (int32, int64) or real ones (fp32, fp64: hours, degrees), [N, axes] for all samples, [B, N, axes] for each its own, [T, axes] of
packed tokens: any single token can stand anywhere.  Angles are taken in 64 bits and reduced to one turn before they are rounded, so that far
positions lose nothing.  No gradient leads to them.

CUDA tensors in bf16 or fp32 with heads of 8, 16, .. 256 channels run on the in-tree kernels (norms' statistics and all sums in fp32, one rounding at the
end); the rest, and what `torch.func`, forward-mode differentiation, tracing or compilation calls, on torch's operations.  A rotation alone can be
differentiated as often as one likes; a graph with norms that the kernels made is differentiated once, and neither in batches of gradients or in a trace.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _ext
from . import attention as attn_ops

AXES = 4               # most axes
WIDTH = 256            # most channels of a head in the kernels
NORMS = {None: 0, "layer": 1, "rms": 2}
_TYPES = (torch.bfloat16, torch.float32)
_POSITIONS = (torch.int32, torch.int64, torch.float32, torch.float64)


class RotaryAxes:
    """How the channels of a head turn: `bands` channels for every axis (even numbers), `base` of the frequencies (one, or one per axis)."""

    def __init__(self, bands: Union[int, Sequence[int]], base: Union[float, Sequence[float]] = 10000.0, interleaved: bool = False):
        bands = (bands,) if isinstance(bands, int) else tuple(bands)
        if not 1 <= len(bands) <= AXES or any(not isinstance(b, int) or isinstance(b, bool) or b < 2 or b % 2 for b in bands):
            raise ValueError(f"rotary positions take one to {AXES} bands of an even number of channels, got {bands}")
        base = (float(base),) * len(bands) if isinstance(base, (int, float)) else tuple(float(b) for b in base)
        if len(base) != len(bands) or any(not (b > 0.0 and math.isfinite(b)) for b in base):
            raise ValueError(f"one positive base, or one for each of {len(bands)} axes expected, got {base}")
        self.bands, self.base, self.interleaved = bands, base, bool(interleaved)
        self.channels = sum(bands)
        # radians per unit of position of every pair
        self.frequencies = [f ** (-2.0 * i / b) for b, f in zip(bands, base) for i in range(b // 2)]
        self._native = None

    def __len__(self) -> int:
        return len(self.bands)

    def __repr__(self) -> str:
        return f"RotaryAxes(bands={self.bands}, base={self.base}, interleaved={self.interleaved})"

    def __eq__(self, other) -> bool:
        return isinstance(other, RotaryAxes) and (self.bands, self.base, self.interleaved) == (other.bands, other.base, other.interleaved)

    def __hash__(self) -> int:
        return hash((self.bands, self.base, self.interleaved))

    def __getstate__(self):
        return {**self.__dict__, "_native": None}

    def native(self):
        if self._native is None:
            self._native = _ext.require().RotaryPlan(list(self.bands), [f / (2.0 * math.pi) for f in self.frequencies], self.interleaved)
        return self._native

    def angles(self, positions: torch.Tensor) -> torch.Tensor:
        """[..., pairs], fp64: what every pair turns by at positions [..., axes]."""
        axis = [a for a, b in enumerate(self.bands) for _ in range(b // 2)]
        f = torch.tensor(self.frequencies, dtype=torch.float64, device=positions.device)
        return positions[..., axis].double() * f


_NO_AXES = None


def _no_axes():
    """The plan of a norm without a rotation."""
    global _NO_AXES
    if _NO_AXES is None:
        _NO_AXES = _ext.require().RotaryPlan([], [], False)
    return _NO_AXES


def grid_positions(*sizes: int, first: int = 0, device=None) -> torch.Tensor:
    """[first + product of sizes, axes], int32: the places of the tokens of a grid, the last axis fastest, behind `first` tokens at the origin."""
    if not sizes or any(s < 1 for s in sizes) or first < 0:
        raise ValueError(f"a grid of at least one token and axis expected, got {sizes} behind {first}")
    axes = torch.meshgrid(*(torch.arange(s, dtype=torch.int32, device=device) for s in sizes), indexing="ij")
    at = torch.stack([a.reshape(-1) for a in axes], -1)
    return torch.cat([at.new_zeros(first, len(sizes)), at]).contiguous()


# ---------------------------------------------------------------------------------------------------- checks

def _check_heads(x, k=None):
    if x.dim() not in (3, 4) or not x.dtype.is_floating_point or x.shape[-1] < 1:
        raise ValueError(f"rotary positions take floating-point tokens [B, N, heads, D] or [T, heads, D], got {x.dtype} {tuple(x.shape)}")
    if k is not None and (k.dim() != x.dim() or k.shape[:-2] != x.shape[:-2] or k.shape[-1] != x.shape[-1] or k.dtype != x.dtype or k.device != x.device):
        raise ValueError(f"queries {x.dtype} {tuple(x.shape)} and keys {k.dtype} {tuple(k.shape)} must be of the same tokens, channels, type and device")


def _check_positions(positions, axes, lead, D, device):
    """Dense positions for tokens [*lead]."""
    if positions is None and axes is None:
        return None
    if positions is None or axes is None:
        raise ValueError("positions and their axes go together")
    if axes.channels > D:
        raise ValueError(f"{axes.channels} channels to turn, heads of {D}")
    if positions.dtype not in _POSITIONS or positions.device != device:
        raise ValueError(f"positions must be int32, int64, fp32 or fp64 on {device}, got {positions.dtype} on {positions.device}")
    if positions.requires_grad:
        raise ValueError("no gradient leads to positions")
    shape = positions.shape
    if not shape or shape[-1] != len(axes.bands) or shape[:-1] != lead and (len(shape) != 2 or shape[0] != lead[-1]):
        raise ValueError(f"positions {tuple(shape)} do not match tokens {tuple(lead)} with {len(axes)} axes")
    return positions.contiguous()


def _check_norm(norm, eps, D, device, params):
    if norm not in NORMS:
        raise ValueError(f"norm must be one of {list(NORMS)}, got {norm!r}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, p in params.items():
        if p is None:
            continue
        if norm is None:
            raise ValueError(f"{name} without a norm")
        if tuple(p.shape) != (D,) or p.device != device or not p.dtype.is_floating_point:
            raise ValueError(f"norm over {D} channels on {device}: {name} is {p.dtype} {tuple(p.shape)} on {p.device}")


def _native(x, D: int) -> bool:
    return _ext.native() and x.is_cuda and x.dtype in _TYPES and D % 8 == 0 and 8 <= D <= WIDTH and not torch.compiler.is_compiling()


# ---------------------------------------------------------------------------------------------------- torch's operations

def _norm_torch(x, weight, bias, eps, norm):
    if norm is None:
        return x
    if norm == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        x = x * weight.to(x.dtype)
    return x if bias is None else x + bias.to(x.dtype)


def _turn_torch(x, positions, axes, inverse):
    if positions is None:
        return x
    angle = axes.angles(positions)[..., None, :]                  # one for all heads
    cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    if inverse:
        sin = -sin
    out, at, pair = [], 0, 0
    for b in axes.bands:
        band, c, s = x[..., at:at + b], cos[..., pair:pair + b // 2], sin[..., pair:pair + b // 2]
        lo, hi = (band[..., 0::2], band[..., 1::2]) if axes.interleaved else band.split(b // 2, -1)
        turned = (lo * c - hi * s, hi * c + lo * s)
        out.append(torch.stack(turned, -1).flatten(-2) if axes.interleaved else torch.cat(turned, -1))
        at, pair = at + b, pair + b // 2
    return torch.cat(out + [x[..., at:]], -1)


def _torch(x, weight, bias, positions, axes, eps, norm, inverse=False):
    device = x.device.type
    if device in ("cuda", "cpu") and torch.is_autocast_enabled(device):
        # (the types are explicit here: autocast would choose its own)
        with torch.autocast(device_type=device, enabled=False):
            return _torch(x, weight, bias, positions, axes, eps, norm, inverse)
    t = torch.promote_types(x.dtype, torch.float32)
    return _turn_torch(_norm_torch(x.to(t), weight, bias, eps, norm), positions, axes, inverse).to(x.dtype)


# ---------------------------------------------------------------------------------------------------- operators

def _kernels(q, k, qw, kw, qb, kb, positions, axes, eps, norm, inverse=False):
    """Results where the tensors are for the kernels and the arguments are in order (the extension looks at them: half of a small call's time went into doing so
    here); else an empty list."""
    if not (_ext.native() and q.is_cuda) or torch.compiler.is_compiling():
        return []
    return _ext.require().rotary_call(q, k, qw, kw, qb, kb, positions, _no_axes() if axes is None else axes.native(), NORMS.get(norm, -1), eps, inverse)


def _run(q, k, qw, kw, qb, kb, positions, axes, eps, norm, inverse=False):
    """Results of one or two tensors whose arguments are checked, in torch's operations."""
    return [_torch(t, w, b, positions, axes, eps, norm, inverse) for t, w, b in ((q, qw, qb), (k, kw, kb)) if t is not None]


def rotary(x: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes, inverse: bool = False) -> torch.Tensor:
    """x [B, N, heads, D] (or [T, heads, D]) turned by its positions, or back with `inverse`; dense, in the type of x."""
    if positions is not None:
        out = _kernels(x, None, None, None, None, None, positions, axes, 0.0, None, bool(inverse))
        if out:
            return out[0]
    _check_heads(x)
    positions = _check_positions(positions, axes, x.shape[:-2], x.shape[-1], x.device)
    if positions is None:
        raise ValueError("rotary takes positions and their axes")
    return _run(x, None, None, None, None, None, positions, axes, 0.0, None, bool(inverse))[0]


def rotary_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries [.., H, D] and keys [.., Hk, D] of the same tokens turned by their positions, in one launch."""
    if positions is not None:
        out = _kernels(q, k, None, None, None, None, positions, axes, 0.0, None)
        if out:
            return out[0], out[1]
    _check_heads(q, k)
    positions = _check_positions(positions, axes, q.shape[:-2], q.shape[-1], q.device)
    if positions is None:
        raise ValueError("rotary_qk takes positions and their axes")
    return tuple(_run(q, k, None, None, None, None, positions, axes, 0.0, None))


def norm_rotary_qk(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                   positions: Optional[torch.Tensor] = None, axes: Optional[RotaryAxes] = None, q_bias: Optional[torch.Tensor] = None,
                   k_bias: Optional[torch.Tensor] = None, eps: float = 1e-5, norm: str = "layer") -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys normed over the channels of every head, then turned, in one pass: `norm` "layer" is (x - mean) / sqrt(var + eps) (biased variance),
    "rms" x / sqrt(mean(x^2) + eps), times weight plus bias ([D] each, or None).  Without positions the norm alone."""
    out = _kernels(q, k, q_weight, k_weight, q_bias, k_bias, positions, axes, float(eps), norm)
    if out and norm is not None:
        return out[0], out[1]
    _check_heads(q, k)
    D = q.shape[-1]
    positions = _check_positions(positions, axes, q.shape[:-2], D, q.device)
    _check_norm(norm, eps, D, q.device, dict(q_weight=q_weight, k_weight=k_weight, q_bias=q_bias, k_bias=k_bias))
    return tuple(_run(q, k, q_weight, k_weight, q_bias, k_bias, positions, axes, float(eps), norm))


def rotary_attention_qkv(qkv: torch.Tensor, num_heads: int, num_kv_heads: Optional[int] = None, positions: Optional[torch.Tensor] = None,
                         axes: Optional[RotaryAxes] = None, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                         q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, eps: float = 1e-5, norm: Optional[str] = None,
                         causal: bool = False, scale: Optional[float] = None, offsets: Optional[torch.Tensor] = None, window: attn_ops.Window = None,
                         sinks: int = 0) -> torch.Tensor:
    """Attention on the output of a fused projection (as `attention.attention_qkv`, with its masks), whose queries and keys are normed (`norm`: "layer", "rms"
    or None) and turned by their positions on the way, in the type of the projection.  The gradient of the projection is written as one tensor:
    attention leaves those of queries and keys where the norm's backward pass replaces them."""
    Hk, D = attn_ops._check_fused(qkv, num_heads, num_kv_heads, offsets)
    packed = offsets is not None
    lead = qkv.shape[:-1]
    positions = _check_positions(positions, axes, lead, D, qkv.device)
    _check_norm(norm, eps, D, qkv.device, dict(q_weight=q_weight, k_weight=k_weight, q_bias=q_bias, k_bias=k_bias))
    if positions is None and norm is None:
        return attn_ops.attention_qkv(qkv, num_heads, num_kv_heads, causal, scale, offsets, window, sinks)
    if _native(qkv, D) and attn_ops.native_ok(qkv, D):
        mask = attn_ops._check_window(window, sinks, causal)
        scale = attn_ops._check_scale(scale, D)
        at = attn_ops._check_offsets(offsets, qkv.shape[0], qkv.device) if packed else None
        o = _ext.require().rotary_attention_qkv(qkv[None] if packed else qkv, num_heads, Hk, q_weight, k_weight, q_bias, k_bias, positions, at,
                                                _no_axes() if axes is None else axes.native(), NORMS[norm], float(eps), causal, scale, *mask)
        if o is not None:
            return o[0] if packed else o
    q, k, v = qkv.unflatten(-1, (num_heads + 2 * Hk, D)).split([num_heads, Hk, Hk], dim=-2)
    # (on the kernels still, where only attention has none: heads of 136 channels, fp32)
    q, k = _kernels(q, k, q_weight, k_weight, q_bias, k_bias, positions, axes, float(eps), norm) or _run(q, k, q_weight, k_weight, q_bias, k_bias, positions, axes, float(eps), norm)
    return attn_ops.attention(q, k, v, causal, scale, offsets, window, sinks)
