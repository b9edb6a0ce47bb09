"""Softmax attention of tokens with themselves, `softmax(scale Q K^T) V`, forward and backward on the tensor cores.

Layout: tokens first, heads inside ([B, N, heads, D]), as a projection writes them and the next one reads them, so that nothing is
transposed.  Grouped heads (`H` of the queries, `Hk` of keys and values, `H % Hk == 0`: query head h reads key head h // (H // Hk)),
causal or not, batches of one length or packed sequences of different lengths.

Packed sequences: tokens [T, heads, D] and `offsets` [S + 1], sequence i is the tokens offsets[i] .. offsets[i + 1]; sequences may be of
one token or of none.  offsets[0] is 0 and none is below the one before it or above T; on the GPU they are read by the kernels and
not checked (out of range they are clamped to it).  Tokens behind offsets[S] belong to no sequence: their outputs and gradients are
zero, and what their inputs hold reaches nothing.

Windows: with `window` a token sees those at most `left` before and `right` behind it (one number: either way; causal: none behind), and with
`sinks` the first tokens of its sequence stay visible from everywhere (causal: from behind them).  Every token sees itself, so that no row is empty.
Tiles that a window leaves out are not visited: the work is that of the window.

bf16 CUDA tensors of up to 128 channels a head run on the in-tree kernels (widths that are no multiple of 8 are padded with zeros);
anything else, and what `torch.func`, forward-mode differentiation, tracing or compilation calls, through torch.  A graph that the
kernels made is differentiated once, and not in batches of gradients or in a trace.  Weights and their gradients are rounded to bf16
where they are operands of the second products; all sums are fp32.  What a causal mask or a window hides has a weight of zero: queries, keys,
values and output gradients of such a sequence have to be finite, or outputs and gradients of tokens that do not see them may be NaN as well.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _ext

WIDTH = 128          # most channels of a head in the kernels


def native_ok(x: torch.Tensor, head_dim: int) -> bool:
    return _ext.native() and x.is_cuda and x.dtype == torch.bfloat16 and 0 < head_dim <= WIDTH and not torch.compiler.is_compiling()


def _check_offsets(offsets, tokens: int, device):
    """int32 offsets on `device`; those that are on the host are checked."""
    if not isinstance(offsets, torch.Tensor):
        offsets = torch.tensor(offsets, dtype=torch.int64)
    if offsets.dim() != 1 or offsets.numel() < 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"offsets must be int32 or int64 [sequences + 1], got {offsets.dtype} {tuple(offsets.shape)}")
    if not offsets.is_cuda:
        at = offsets.tolist()
        if at[0] != 0 or at[-1] > tokens or any(a > b for a, b in zip(at, at[1:])):
            raise ValueError(f"offsets must rise from 0 to at most the {tokens} tokens, got {at}")
    elif offsets.device != device:
        raise ValueError(f"offsets on {offsets.device}, tokens on {device}")
    return offsets.to(device=device, dtype=torch.int32).contiguous()


def _check_scale(scale, head_dim: int) -> float:
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"attention takes a positive scale, got {scale}")
    return scale


Window = Union[None, int, Tuple[Optional[int], Optional[int]]]


def _check_window(window: Window, sinks: int, causal: bool):
    """(left, right, sinks), -1 for no end; (-1, -1, 0): everything is visible."""
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise ValueError(f"sinks must be a number of tokens, got {sinks!r}")
    if window is None:
        return -1, -1, 0
    pair = (window, window) if isinstance(window, int) and not isinstance(window, bool) else window
    if not isinstance(pair, (tuple, list)) or len(pair) != 2 or any(w is not None and (isinstance(w, bool) or not isinstance(w, int) or w < 0) for w in pair):
        raise ValueError(f"a window is a number of tokens, or (left, right) of them or None, got {window!r}")
    left, right = (-1 if w is None else w for w in pair)
    if left < 0 and (causal or right < 0):
        return -1, -1, 0
    return left, 0 if causal else right, sinks


def visible(tokens: int, causal: bool = False, window: Window = None, sinks: int = 0, device=None) -> torch.Tensor:
    """[tokens, tokens], boolean: whether a query (row) sees a key (column) of one sequence."""
    left, right, sinks = _check_window(window, sinks, causal)
    return _visible(torch.arange(tokens, device=device), tokens, causal, left, right, sinks)


def _visible(i, tokens, causal, left, right, sinks):
    j = torch.arange(tokens, device=i.device)
    away = i[:, None] - j[None, :]
    seen = torch.ones_like(away, dtype=torch.bool)
    if left >= 0:
        seen &= away <= left
    if right >= 0:
        seen &= away >= -right
    if sinks > 0:
        seen |= j[None, :] < sinks
    if causal:
        seen &= away >= 0
    return seen


QUERIES_AT_ONCE = 1024      # of a windowed pass through the library, whose mask is a tensor


def _attend_torch(q, k, v, causal, scale, offsets=None, mask=(-1, -1, 0)):
    """[B, N, heads, D], or packed [T, heads, D], through the library."""
    if offsets is not None:
        at = offsets.tolist()
        # (an empty sequence in front: with nothing behind it the result is still a function of the inputs)
        parts = [_attend_torch(*(t[None, a:b] for t in (q, k, v)), causal, scale, None, mask)[0] for a, b in [(0, 0)] + [r for r in zip(at, at[1:]) if r[1] > r[0]]]
        return torch.cat(parts + [torch.zeros_like(q[at[-1]:])])
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    if k.shape[1] != q.shape[1]:
        k, v = (t.repeat_interleave(int(q.shape[1] // t.shape[1]), dim=1) for t in (k, v))      # (a trace has tensors for sizes)
    sdpa = torch.nn.functional.scaled_dot_product_attention
    if mask[0] < 0 and mask[1] < 0:
        return sdpa(q, k, v, is_causal=causal, scale=scale).transpose(1, 2).contiguous()
    N = q.shape[2]
    parts = []
    for lo in range(0, max(N, 1), QUERIES_AT_ONCE):
        hi = min(N, lo + QUERIES_AT_ONCE)
        seen = _visible(torch.arange(lo, hi, device=q.device), N, causal, *mask)
        parts.append(sdpa(q[:, :, lo:hi], k, v, attn_mask=seen, scale=scale))
    return torch.cat(parts, 2).transpose(1, 2).contiguous()


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = False, scale: Optional[float] = None,
              offsets: Optional[torch.Tensor] = None, window: Window = None, sinks: int = 0) -> torch.Tensor:
    """softmax(scale q k^T) v per head: q [B, N, H, D], k and v [B, N, Hk, D], or packed [T, H, D] with `offsets`; the result is like q,
    dense.  `scale` defaults to D ** -0.5; `window` and `sinks` as above."""
    if _ext.native() and q.is_cuda and (offsets is None or isinstance(offsets, torch.Tensor)) and not torch.compiler.is_compiling():
        # (what is for the kernels and in order needs no closer look)
        o = _ext.require().attention_call(q, k, v, offsets, causal, scale, *_check_window(window, sinks, causal))
        if o is not None:
            return o
    packed = offsets is not None
    if not (q.dim() == k.dim() == v.dim() == (3 if packed else 4)):
        raise ValueError(f"attention takes {'[T, heads, D] with' if packed else '[B, N, heads, D] without'} offsets, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape != v.shape or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"queries {tuple(q.shape)}, keys {tuple(k.shape)} and values {tuple(v.shape)} must be of the same tokens and channels")
    if q.shape[-2] < 1 or k.shape[-2] < 1 or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"{q.shape[-2]} heads of queries, {k.shape[-2]} of keys: there must be some, and those of keys divide those of queries")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device and q.dtype.is_floating_point):
        raise ValueError("queries, keys and values must share one floating-point type and device")
    if q.shape[-1] < 1:
        raise ValueError("heads without channels")
    D = q.shape[-1]
    scale = _check_scale(scale, D)
    mask = _check_window(window, sinks, causal)
    if packed:
        offsets = _check_offsets(offsets, q.shape[0], q.device)
    if not native_ok(q, D):
        return _attend_torch(q, k, v, causal, scale, offsets, mask)
    views = (t[None] for t in (q, k, v)) if packed else (q, k, v)
    more = -D % 8
    if more:
        views = (torch.nn.functional.pad(t, (0, more)) for t in views)
    o = _ext.require().attention(*views, offsets, causal, scale, *mask)
    if o is None:      # (the call is a transform's, a trace's or a mode's)
        return _attend_torch(q, k, v, causal, scale, offsets, mask)
    if more:
        o = o[..., :D].contiguous()
    return o[0] if packed else o


def _check_fused(qkv, num_heads, num_kv_heads, offsets):
    """(heads of keys, channels of a head) of a fused projection's output."""
    Hk = num_heads if num_kv_heads is None else num_kv_heads
    packed = offsets is not None
    if qkv.dim() != (2 if packed else 3) or not qkv.dtype.is_floating_point:
        raise ValueError(f"attention_qkv takes {'[T, channels] with' if packed else '[B, N, channels] without'} offsets, got {qkv.dtype} {tuple(qkv.shape)}")
    if num_heads < 1 or Hk < 1 or num_heads % Hk:
        raise ValueError(f"{Hk} heads of keys do not divide {num_heads} of queries")
    if qkv.shape[-1] < 1 or qkv.shape[-1] % (num_heads + 2 * Hk):
        raise ValueError(f"{qkv.shape[-1]} channels are not those of {num_heads} + 2 x {Hk} heads")
    return Hk, qkv.shape[-1] // (num_heads + 2 * Hk)


def attention_qkv(qkv: torch.Tensor, num_heads: int, num_kv_heads: Optional[int] = None, causal: bool = False, scale: Optional[float] = None,
                  offsets: Optional[torch.Tensor] = None, window: Window = None, sinks: int = 0) -> torch.Tensor:
    """`attention` on the output of a fused projection, [B, N, (H + 2 Hk) * D] (or packed [T, ...] with `offsets`): the channels of all
    queries' heads, then those of the keys' and of the values'.  Returns [B, N, H, D] ([T, H, D]); the gradient is one tensor like `qkv`."""
    Hk, D = _check_fused(qkv, num_heads, num_kv_heads, offsets)
    packed = offsets is not None
    mask = _check_window(window, sinks, causal)
    if native_ok(qkv, D) and D % 8 == 0:
        scale = _check_scale(scale, D)
        if packed:
            offsets = _check_offsets(offsets, qkv.shape[0], qkv.device)
        o = _ext.require().attention_qkv(qkv[None] if packed else qkv, num_heads, Hk, offsets, causal, scale, *mask)
        if o is not None:
            return o[0] if packed else o
    if Hk == num_heads and not packed and mask == (-1, -1, 0):      # (views of one tensor, heads in front, whose gradient is one copy)
        scale = _check_scale(scale, D)
        q, k, v = qkv.reshape(*qkv.shape[:-1], 3, num_heads, D).permute(2, 0, 3, 1, 4).unbind(0)
        return torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=causal, scale=scale).transpose(1, 2).contiguous()
    q, k, v = qkv.unflatten(-1, (num_heads + 2 * Hk, D)).split([num_heads, Hk, Hk], dim=-2)
    return attention(q, k, v, causal, scale, offsets, window, sinks)
