"""Dropout with an added residual whose mask is never stored: y = residual + x * keep / (1 - p), dx = dy * keep / (1 - p).

``keep`` of an element is a function of (seed, site, row, column) alone: 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) at counter
(column // 8, row % 2^32, row // 2^32, site) and key (seed % 2^32, seed // 2^32); column c takes half c % 8 of the four words, low halves first, and is
kept where that half is at least round(65536 p). p is met to 2^-17 and the scale fits the p that is used. So a checkpointed layer that runs again in
the backward pass drops what it dropped, and ranks that hold some of the rows each (``row0`` = their first one) together drop what one rank would.

``seed``: an int of 0 to 2^64 - 1, or an int64 tensor of one element on the device (a captured graph then reads a new seed at every replay).
``site`` (0 to 2^32 - 1) tells the places of a model apart. What stands in dropped places of ``x`` does not matter. Tensors are bf16 or fp32
[rows, cols], rows may be strided; GPU tensors use csrc/cuda/dropout.cu, CPU tensors the same arithmetic in PyTorch.
"""
from __future__ import annotations

import torch

from .._lib import ptr
from .launch import launch, refuse_capture, rows_of

_DTYPES = (torch.bfloat16, torch.float32)


def threshold_of(p: float) -> int:
    """Values of 16 bits that drop an element."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p}: 0 to 1 is wanted")
    return int(round(p * 65536))


def _scale_of(t: int) -> float:
    return 65536.0 / (65536 - t) if t < 65536 else 0.0


def _check(x, seed, row0, site, residual=None):
    allowed = _DTYPES if x.is_cuda else _DTYPES + (torch.float64,)
    if x.dim() != 2:
        raise ValueError(f"rows [rows, cols] are wanted: got {tuple(x.shape)}")
    if x.dtype not in allowed:
        raise TypeError(f"rows of type {x.dtype}: bf16 and fp32 are supported")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} on {residual.device} for rows {tuple(x.shape)} {x.dtype} on {x.device}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError(f"a seed tensor is one int64 element on {x.device}: got {tuple(seed.shape)} {seed.dtype} on {seed.device}")
    elif not 0 <= seed < 1 << 64:
        raise ValueError(f"seed {seed}: 0 to 2^64 - 1 is wanted")
    if not 0 <= row0 <= (1 << 63) - 1 - x.shape[0]:
        raise ValueError(f"row0 {row0}: zero or a positive number below 2^63 is wanted")
    if not 0 <= site < 1 << 32:
        raise ValueError(f"site {site}: 0 to 2^32 - 1 is wanted")


def philox4x32(counter, key):
    """Philox4x32-10 on int64 tensors that hold 32-bit words: four words for each counter of four words."""
    c0, c1, c2, c3 = counter
    k0, k1 = key
    low = 0xFFFFFFFF
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def keep_mask(rows: int, cols: int, p: float, seed: int, row0: int = 0, site: int = 0) -> torch.Tensor:
    """The mask, bool [rows, cols] on the CPU."""
    n = (cols + 7) // 8
    row = (torch.arange(rows, dtype=torch.int64) + row0)[:, None].expand(rows, n)
    group = torch.arange(n, dtype=torch.int64)[None].expand(rows, n)
    seed = int(seed) & (1 << 64) - 1
    words = philox4x32((group, row & 0xFFFFFFFF, row >> 32, torch.full_like(row, site)), (seed & 0xFFFFFFFF, seed >> 32))
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], -1).reshape(rows, n * 8)[:, :cols]
    return halves >= threshold_of(p)


def _launch(x, residual, t, seed, row0, site):
    x = rows_of(x)
    residual = rows_of(residual) if residual is not None else None
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    on_device = isinstance(seed, torch.Tensor)
    launch(x.device, "dropout", "plplpiliiflpli", x.data_ptr(), x.stride(0), ptr(residual), residual.stride(0) if residual is not None else 0, y.data_ptr(),
           x.dtype == torch.float32, x.shape[0], x.shape[1], t, _scale_of(t), 0 if on_device else seed, seed.data_ptr() if on_device else 0, row0, site)
    return y


def _plain(x, residual, p, seed, row0, site):
    t = threshold_of(p)
    keep = keep_mask(x.shape[0], x.shape[1], p, int(seed), row0, site)
    wide = x if x.dtype == torch.float64 else x.float()
    y = torch.where(keep, wide * _scale_of(t), torch.zeros((), dtype=wide.dtype))
    if residual is not None:
        y = y + residual.to(wide.dtype)
    return y.to(x.dtype)


def dropout_add(x, p: float, seed, *, residual=None, row0: int = 0, site: int = 0):
    """residual + dropout(x) (dropout(x) without a residual), rounded once."""
    _check(x, seed, row0, site, residual)
    t = threshold_of(p)
    return _launch(x, residual, t, seed, row0, site) if x.is_cuda else _plain(x, residual, p, seed, row0, site)


def dropout_backward(dy, p: float, seed, *, row0: int = 0, site: int = 0):
    """Gradient of ``x`` in ``dropout_add`` with the same p, seed, row0 and site (that of the residual is ``dy``)."""
    return dropout_add(dy, p, seed, row0=row0, site=site)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, row0, site):
        refuse_capture(x)
        tensor = isinstance(seed, torch.Tensor)
        if tensor:
            ctx.save_for_backward(seed)            # (changed before the backward pass: autograd says so)
        ctx.args = (p, None if tensor else seed, row0, site)
        return dropout_add(x, p, seed, residual=residual, row0=row0, site=site)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        refuse_capture(dy)
        p, seed, row0, site = ctx.args
        if seed is None:
            (seed,) = ctx.saved_tensors
        dx = dropout_backward(dy, p, seed, row0=row0, site=site) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout_residual(x, p: float, seed, residual=None, row0: int = 0, site: int = 0):
    """``dropout_add``, differentiable in ``x`` and ``residual``."""
    return _DropoutAdd.apply(x, residual, p, seed, row0, site)
