"""Dropout whose mask is a function of a seed and the element, made again in the backward pass and never stored; alone, or with a residual sum behind it.

Element i, in the order of a dense tensor, is kept if its 32 random bits, as a number, are at least p 2^32: word i % 4 of the Philox4x32 generator of ten
rounds (Salmon et al., 2011) whose counter is (number of the call, i // 4), 64 bits each, and whose key is the seed.  What is kept is divided by 1 - p,
what is dropped is zero, whatever it was.

`seed` is an int64 tensor (key, number of the call) on the device of x; two calls with the same draw the same mask, on any device.  Without it the
generator is torch's of the device: `torch.manual_seed`, `torch.random.fork_rng`, checkpointing and captured graphs, whose replays draw new masks, work
as with torch's own dropout (whose masks are others).

bf16 and fp32 CUDA tensors run on the in-tree kernel; the rest, and what `torch.func`, forward-mode differentiation, tracing or compilation calls, on
torch's operations.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _ext


def _check(x, p, seed, residual=None):
    if not x.dtype.is_floating_point:
        raise ValueError(f"dropout takes floating-point tensors, got {x.dtype}")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout takes a probability, got {p}")
    if residual is not None and (residual.shape != x.shape or residual.device != x.device or not residual.dtype.is_floating_point):
        raise ValueError(f"the residual {residual.dtype} {tuple(residual.shape)} on {residual.device} does not match {tuple(x.shape)} on {x.device}")
    if seed is not None and (seed.dtype != torch.int64 or seed.numel() != 2 or seed.dim() != 1 or seed.device != x.device):
        raise ValueError(f"a seed is two int64 on {x.device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")


def random_words(seed: torch.Tensor, n: int) -> torch.Tensor:
    """The 32 random bits of elements 0 .. n - 1 of a call, int64, in torch's operations on the device of `seed`."""
    m = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, dtype=torch.int64, device=seed.device)
    key, number = seed[0], seed[1].expand_as(block)
    c0, c1, c2, c3 = number & m, (number >> 32) & m, block & m, block >> 32
    k0, k1 = key & m, (key >> 32) & m
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # (64 bits, wrapped: both halves are right)
        c0, c1, c2, c3 = ((p1 >> 32) & m) ^ c1 ^ k0, p1 & m, ((p0 >> 32) & m) ^ c3 ^ k1, p0 & m
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return torch.stack([c0, c1, c2, c3], -1).flatten()[:n]


def _dropped_torch(x, p, seed):
    if seed is None:
        return torch.nn.functional.dropout(x, p, True)
    keep = (random_words(seed, x.numel()) >= round(p * 2 ** 32)).view(x.shape)
    t = torch.promote_types(x.dtype, torch.float32)
    return torch.where(keep, x.to(t) / (1.0 - p) if p < 1.0 else x.to(t), torch.zeros((), dtype=t, device=x.device))


def _kernel(x, residual, p, seed):
    """The result where the tensors are for the kernel and the arguments are in order (the extension looks at them); else None."""
    if not (_ext.native() and x.is_cuda) or torch.compiler.is_compiling():
        return None
    return _ext.require().dropout_call(x, residual, seed, p)


LEAST = 2.0 ** -33          # p that rounds to no word of 2^32


def dropout(x: torch.Tensor, p: float = 0.5, training: bool = True, seed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x / (1 - p) where an element is kept, zero where it is dropped; x itself where nothing is to be dropped."""
    if training and p > LEAST:
        y = _kernel(x, None, p, seed)
        if y is not None:      # (None: the call is a transform's, a trace's or a mode's, too)
            return y
    _check(x, p, seed)
    if not training or p <= LEAST:
        return x
    return _dropped_torch(x, p, seed).to(x.dtype)


def dropout_add(x: torch.Tensor, residual: torch.Tensor, p: float = 0.5, training: bool = True, seed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dropout(x) + residual, in the wider of their types, rounded once; one pass over memory in either direction."""
    if training and p > LEAST:
        y = _kernel(x, residual, p, seed)
        if y is not None:
            return y
    _check(x, p, seed, residual)
    if not training or p <= LEAST:
        return x + residual
    t = torch.promote_types(x.dtype, residual.dtype)
    wide = torch.promote_types(t, torch.float32)
    return (_dropped_torch(x.to(wide), p, seed) + residual.to(wide)).to(t)
