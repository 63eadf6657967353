"""Losses of a language model head that never hold its logits: softmax cross entropy against labels, and KL(teacher || model) against a teacher's
K most likely tokens and the mass of the rest (what ``volta_ppl --topk-out`` writes); both with the gradients of the states and of the head.

    z = cap(x head^T),  cap(z) = softcap * tanh(z / softcap) (softcap 0: z as it is)        s = softmax(z)
    cross entropy   nll = log sum_v exp z_v - z_label
    divergence      kl  = sum_k a_k (log a_k - log s_k) + t (log t - log max(r, 1e-12)),  a = exp(logp), t = exp(tail),
                    r = the model's mass outside the teacher's tokens, k over the tokens that the teacher lists

``x`` [rows, hidden] and ``head`` [vocab, hidden] are bf16 or fp32, each by itself; sums are 32 bits wide and the products of fp32 operands exact to
2^-24. Rows may be strided. Losses and their sums are fp32; dx has the type of x, dhead that of head.

Rows that do not count: a negative label, or a teacher row whose ids are all negative (single negative ids are padding). Their loss, statistics and
gradients are zero and their states are not read. An id listed twice is one token whose teacher's mass is the sum. A label or id at or behind
``vocab`` makes the row's loss NaN (and with it the gradients it takes part in): the ids stay on the device, nothing waits to look at them. NaN among a
row's logits or its teacher's numbers is its loss.

GPU tensors use csrc/cuda/head_loss.cu: the explicit forward / backward pairs launch on the current stream of the tensors' device, take their
workspace from the caching allocator and may be captured into a CUDA graph. The same call gives the same bits; between calls of few and of many rows the last
bits of a row's loss may differ (sums of exponentials by blocks of 32 tokens, or of 128). CPU tensors run the same arithmetic in PyTorch (fp64 stays fp64).
``head_cross_entropy_loss`` and ``head_kl_loss`` are the pairs as one differentiable call.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch

from .._lib import kernels, ptr
from ..ops.kernels import status_word
from .launch import launch, refuse_capture, rows_of

MAX_TOPK = 1024
REST_FLOOR = 1e-12                 # least probability of "any other token" in a divergence
_DTYPES = (torch.bfloat16, torch.float32)


# ------------------------------------------------------------------------------------------------ arguments
def _check(x, head, softcap, others, dloss=None, stats=None):
    """Shapes, types and devices of a call; ``others``: (name, tensor, dtypes, shape)."""
    if x.dim() != 2 or head.dim() != 2 or x.shape[1] != head.shape[1]:
        raise ValueError(f"states [rows, hidden] and head [vocab, hidden] are wanted: got {tuple(x.shape)} and {tuple(head.shape)}")
    rows, vocab, device = x.shape[0], head.shape[0], x.device
    if vocab < 1 or x.shape[1] < 1:
        raise ValueError(f"a head of {tuple(head.shape)} has no logits")
    if rows > (1 << 24) - 256 or vocab >= 1 << 24:            # (rows are padded to whole tiles of 256)
        raise ValueError("rows have to stay below 2^24 - 255, the vocabulary below 2^24")
    allowed = _DTYPES if x.is_cuda else _DTYPES + (torch.float64,)
    if x.dtype not in allowed:
        raise TypeError(f"states of type {x.dtype}: bf16 and fp32 are supported")
    if head.dtype not in allowed:
        raise TypeError(f"head of type {head.dtype}: bf16 and fp32 are supported")
    if head.device != device:
        raise ValueError(f"head on {head.device}, states on {device}")
    if softcap != 0 and not 1e-30 <= softcap < math.inf:
        raise ValueError(f"softcap {softcap}: zero (none) or a number of at least 1e-30 is wanted")
    if dloss is not None:
        f = (torch.float32,) if x.is_cuda else (torch.float32, torch.float64)
        others += (("dloss", dloss, f, (rows,)), ("stats", stats, f, (4 if stats.shape[:1] == (4,) else 2, rows)))
    for name, t, dtypes, shape in others:
        if t.dtype not in dtypes:
            raise TypeError(f"{name} of type {t.dtype}: {' or '.join(str(d) for d in dtypes)} is wanted")
        if t.shape != shape:
            raise ValueError(f"{name} of shape {tuple(t.shape)}: {shape} is wanted")
        if t.device != device:
            raise ValueError(f"{name} on {t.device}, states on {device}")


def _label_args(x, labels):
    return (("labels", labels, (torch.int64, torch.int32), (x.shape[0],)),)


def _teacher_args(x, ids, logp, tail):
    if ids.dim() != 2 or not 1 <= ids.shape[1] <= MAX_TOPK:
        raise ValueError(f"teacher ids [rows, K] with K of 1 to {MAX_TOPK} are wanted: got {tuple(ids.shape)}")
    f = (torch.float32,) if x.is_cuda else (torch.float32, torch.float64)
    rows, k = x.shape[0], ids.shape[1]
    return ("ids", ids, (torch.int32,), (rows, k)), ("logp", logp, f, (rows, k)), ("tail", tail, f, (rows,))


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes) -> int:
    fn = kernels().ve_head_loss_workspace
    fn.argtypes = [ctypes.c_int] * 10
    fn.restype = ctypes.c_int64
    return fn(*sizes)


def _workspace(grads, want_dx, x, head, K, kl):
    packs = head.dtype == torch.float32 or head.shape[1] % 8 != 0 or head.stride(0) % 8 != 0 or head.data_ptr() % 16 != 0
    n = _workspace_bytes(grads, want_dx, x.dtype == torch.float32, head.dtype == torch.float32, packs, x.shape[0], x.shape[1], head.shape[0], K, kl)
    return torch.empty(n, dtype=torch.uint8, device=x.device)


_SIG = "pilpilpipppiiiif"


def _common(x, head, labels, teacher, softcap):
    ids, logp, tail = teacher or (None, None, None)
    return (x.data_ptr(), x.dtype == torch.float32, x.stride(0), head.data_ptr(), head.dtype == torch.float32, head.stride(0), ptr(labels),
            labels.element_size() if labels is not None else 0, ptr(ids), ptr(logp), ptr(tail), ids.shape[1] if teacher else 1, x.shape[0], x.shape[1],
            head.shape[0], softcap)


def _forward(x, head, labels, teacher, softcap, fine):
    x, head = rows_of(x), rows_of(head)
    rows = x.shape[0]
    teacher = tuple(t.contiguous() for t in teacher) if teacher else None
    labels = labels.contiguous() if labels is not None else None
    out = torch.empty(5 if fine else 3, rows, dtype=torch.float32, device=x.device)
    loss, stats = out[0], out[1:]
    if rows:
        ws = _workspace(False, False, x, head, teacher[0].shape[1] if teacher else 1, teacher is not None)
        launch(x.device, "head_loss", _SIG + "ppiplp", *_common(x, head, labels, teacher, softcap), loss.data_ptr(), stats.data_ptr(), fine, ws.data_ptr(),
               ws.numel(), status_word(x.device).data_ptr())
    return loss, stats


def _backward(x, head, labels, teacher, stats, dloss, softcap, want_dx, want_dhead):
    x, head = rows_of(x), rows_of(head)
    rows = x.shape[0]
    teacher = tuple(t.contiguous() for t in teacher) if teacher else None
    labels = labels.contiguous() if labels is not None else None
    stats, dloss = stats.contiguous(), dloss.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_dx else None
    dhead = (torch.empty if rows else torch.zeros)(head.shape, dtype=head.dtype, device=x.device) if want_dhead else None
    if rows:
        ws = _workspace(True, want_dx, x, head, teacher[0].shape[1] if teacher else 1, teacher is not None)
        launch(x.device, "head_loss_grad", _SIG + "pipppplp", *_common(x, head, labels, teacher, softcap), stats.data_ptr(), stats.shape[0] == 4,
               dloss.data_ptr(), ptr(dx), ptr(dhead), ws.data_ptr(), ws.numel(), status_word(x.device).data_ptr())
    return dx, dhead


# ------------------------------------------------------------------------------------------------ the statement in PyTorch (CPU)
def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _capped(x, head, softcap):
    z = _wide(x) @ _wide(head).t()
    if softcap > 0:
        t = torch.tanh(z / softcap)
        return softcap * t, 1 - t * t
    return z, None


def _gathered(x, live):
    """The rows that count (what stands in the others is not used)."""
    return x[live] if not bool(live.all()) else x


def _spread(v, live):
    out = torch.zeros(live.shape[0], *v.shape[1:], dtype=v.dtype)
    out[live] = v
    return out


def _sums(z, targets):
    """-> (log sum exp, the same without ``targets``), targets bool [rows, vocab]."""
    return torch.logsumexp(z, 1), torch.logsumexp(z.masked_fill(targets, -math.inf), 1)


def _stats_out(lse, rest, live, fine):
    out = torch.stack([_spread(lse, live), _spread(rest, live)])
    return torch.cat([out, torch.zeros_like(out)]) if fine else out                # (sums in the states' own width: nothing behind them)


def _stats_in(stats, live, dtype):
    s = stats.to(dtype)[:, live]
    return s[:2] + s[2:] if s.shape[0] == 4 else s


def _finish_grads(dz, slope, bad, x, head, live, want_dx, want_dhead):
    if slope is not None:
        dz = dz * slope
    dz = torch.where(bad[:, None], torch.full_like(dz, math.nan), dz)
    dx = _spread((dz @ _wide(head)).to(x.dtype), live) if want_dx else None
    dhead = (dz.t() @ _wide(_gathered(x, live))).to(head.dtype) if want_dhead else None
    return dx, dhead


def _cpu_labels(z, labels):
    bad = labels >= z.shape[1]
    y = labels.long().clamp(max=z.shape[1] - 1)[:, None]
    return bad, y, torch.zeros_like(z, dtype=torch.bool).scatter_(1, y, True)


def _cpu_ce(x, head, labels, softcap, fine):
    live = labels >= 0
    z, _ = _capped(_gathered(x, live), head, softcap)
    bad, y, hit = _cpu_labels(z, labels[live])
    lse, rest = _sums(z, hit)
    nll = torch.nn.functional.softplus(rest - z.gather(1, y)[:, 0], threshold=1e9)
    nan = torch.full_like(nll, math.nan)
    return _spread(torch.where(bad, nan, nll), live), _stats_out(torch.where(bad, nan, lse), rest, live, fine)


def _cpu_ce_grad(x, head, labels, stats, dloss, softcap, want_dx, want_dhead):
    live = labels >= 0
    z, slope = _capped(_gathered(x, live), head, softcap)
    bad, y, _ = _cpu_labels(z, labels[live])
    lse, rest = _stats_in(stats, live, z.dtype)
    dz = torch.exp(z - lse[:, None]).scatter(1, y, -torch.exp(rest - lse)[:, None]) * dloss[live].to(z.dtype)[:, None]
    return _finish_grads(dz, slope, bad, x, head, live, want_dx, want_dhead)


def _cpu_teacher(z, ids, logp, tail):
    """-> (bad rows, places, the teacher's masses with zeros at padding, log masses, rest mass, targets bool)."""
    vocab = z.shape[1]
    known, at = ids >= 0, ids.long().clamp(0, vocab - 1)
    bad = ((ids >= vocab) & known).any(1)
    hit = torch.zeros(z.shape[0], vocab + 1, dtype=torch.bool).scatter_(1, torch.where(known & (ids < vocab), ids.long(), vocab), True)[:, :vocab]
    logp = torch.where(known, logp.to(z.dtype), torch.full((), -math.inf, dtype=z.dtype))
    return bad, at, torch.exp(logp), logp, tail.to(z.dtype), hit


def _cpu_kl(x, head, ids, logp, tail, softcap, fine):
    live = (ids >= 0).any(1)
    z, _ = _capped(_gathered(x, live), head, softcap)
    bad, at, a, logp, tail, hit = _cpu_teacher(z, ids[live], logp[live], tail[live])
    lse, rest = _sums(z, hit)
    zero = torch.zeros((), dtype=z.dtype)
    whole = torch.zeros_like(z).scatter_add_(1, at, a).gather(1, at)             # the mass of an entry's token (more than its own where it is listed again)
    kl = torch.where(a == 0, zero, a * (torch.where(whole > a, torch.log(whole), logp) - (z.gather(1, at) - lse[:, None]))).sum(1)
    kl = kl + torch.where(tail == -math.inf, zero, torch.exp(tail) * (tail - (rest - lse).clamp(min=math.log(REST_FLOOR))))
    nan = torch.full_like(kl, math.nan)
    return _spread(torch.where(bad, nan, kl), live), _stats_out(torch.where(bad, nan, lse), rest, live, fine)


def _cpu_kl_grad(x, head, ids, logp, tail, stats, dloss, softcap, want_dx, want_dhead):
    live = (ids >= 0).any(1)
    z, slope = _capped(_gathered(x, live), head, softcap)
    bad, at, a, _, tail, hit = _cpu_teacher(z, ids[live], logp[live], tail[live])
    lse, rest = _stats_in(stats, live, z.dtype)
    s, t = torch.exp(z - lse[:, None]), torch.exp(tail)
    t = torch.where(rest - lse >= math.log(REST_FLOOR), t, torch.zeros_like(t))
    over = torch.where(t > 0, t * torch.exp(lse - rest), t)
    dz = s * (a.sum(1) + t)[:, None] - s.masked_fill(hit, 0.0) * over[:, None]
    dz = dz.scatter_add(1, at, -a) * dloss[live].to(z.dtype)[:, None]
    return _finish_grads(dz, slope, bad, x, head, live, want_dx, want_dhead)


# ------------------------------------------------------------------------------------------------ entry points
def head_cross_entropy(x, head, labels, *, softcap: float = 0.0, fine: bool = False):
    """-> (nll [rows], stats [2, rows]): stats are log sum_v exp z_v and the same sum without the label, for the backward pass. ``fine``: stats [4, rows],
    behind both what their rounding to 32 bits left. The backward pass takes either; a sum of 16 to 32 is off by up to 2^-20 without, which a row's
    gradients have in common: fp32 gradients of few rows, and those of a model near its teacher, are more exact with it."""
    _check(x, head, softcap, _label_args(x, labels))
    return _forward(x, head, labels, None, softcap, fine) if x.is_cuda else _cpu_ce(x, head, labels, softcap, fine)


def head_cross_entropy_backward(x, head, labels, stats, dloss, *, softcap: float = 0.0, want_dx: bool = True, want_dhead: bool = True):
    """Gradients of ``(nll * dloss).sum()``: -> (dx or None, dhead or None)."""
    _check(x, head, softcap, _label_args(x, labels), dloss, stats)
    if not (want_dx or want_dhead):
        return None, None
    if x.is_cuda:
        return _backward(x, head, labels, None, stats, dloss, softcap, want_dx, want_dhead)
    return _cpu_ce_grad(x, head, labels, stats, dloss, softcap, want_dx, want_dhead)


def head_kl(x, head, ids, logp, tail, *, softcap: float = 0.0, fine: bool = False):
    """ids int32 [rows, K], logp fp32 [rows, K] and tail fp32 [rows]: the teacher's tokens, their log-probabilities and the log of the mass outside
    them. -> (kl [rows], stats [2, rows]): stats are log sum_v exp z_v and the same sum without the teacher's tokens (``fine``: as
    ``head_cross_entropy``'s)."""
    _check(x, head, softcap, _teacher_args(x, ids, logp, tail))
    return _forward(x, head, None, (ids, logp, tail), softcap, fine) if x.is_cuda else _cpu_kl(x, head, ids, logp, tail, softcap, fine)


def head_kl_backward(x, head, ids, logp, tail, stats, dloss, *, softcap: float = 0.0, want_dx: bool = True, want_dhead: bool = True):
    """Gradients of ``(kl * dloss).sum()``: -> (dx or None, dhead or None). The teacher is a constant."""
    _check(x, head, softcap, _teacher_args(x, ids, logp, tail), dloss, stats)
    if not (want_dx or want_dhead):
        return None, None
    if x.is_cuda:
        return _backward(x, head, None, (ids, logp, tail), stats, dloss, softcap, want_dx, want_dhead)
    return _cpu_kl_grad(x, head, ids, logp, tail, stats, dloss, softcap, want_dx, want_dhead)


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, head, softcap, fine, *targets):
        refuse_capture(x)
        loss, stats = (head_cross_entropy if len(targets) == 1 else head_kl)(x, head, *targets, softcap=softcap, fine=fine)
        ctx.save_for_backward(x, head, stats, *targets)
        ctx.softcap = softcap
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, head, stats, *targets = ctx.saved_tensors
        refuse_capture(x)
        fn = head_cross_entropy_backward if len(targets) == 1 else head_kl_backward
        dx, dhead = fn(x, head, *targets, stats, dloss.to(stats.dtype), softcap=ctx.softcap, want_dx=ctx.needs_input_grad[0],
                       want_dhead=ctx.needs_input_grad[1])
        return (dx, dhead, None, None) + (None,) * len(targets)


def head_cross_entropy_loss(x, head, labels, softcap: float = 0.0, fine: bool = False):
    """nll [rows], differentiable in ``x`` and ``head``; ``fine`` as in ``head_cross_entropy``."""
    return _HeadLoss.apply(x, head, float(softcap), fine, labels)


def head_kl_loss(x, head, ids, logp, tail, softcap: float = 0.0, fine: bool = False):
    """kl [rows], differentiable in ``x`` and ``head``; ``fine`` as in ``head_cross_entropy``."""
    return _HeadLoss.apply(x, head, float(softcap), fine, ids, logp, tail)
