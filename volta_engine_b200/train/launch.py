"""What the training operators share when they launch: the tensors' device, rows in place, and the differentiable calls' stand on graph capture."""
from __future__ import annotations

import torch

from .._lib import call_on


def launch(device, name: str, sig: str, *args) -> None:
    """``ve_<name>`` on ``device`` and its current stream, whichever device is current."""
    stream = torch._C._cuda_getCurrentRawStream(device.index)           # (the handle alone: a Stream object costs more than a small kernel)
    if device.index == torch._C._cuda_getDevice():
        call_on(stream, name, sig, *args)
    else:
        with torch.cuda.device(device):
            call_on(stream, name, sig, *args)


def rows_of(t):
    """A matrix whose rows' elements lie side by side: ``t`` itself where they do."""
    if t.stride(1) == 1 and t.stride(0) >= t.shape[1] or t.shape[0] == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)          # (``contiguous`` leaves the pitch of a single row as it is, zero for an expanded one)


def refuse_capture(t):
    """Differentiable calls are not captured: a captured backward pass that meets leaves of an eager graph joins streams outside the capture, and the
    process ends. The explicit forward and backward functions may be captured."""
    if t.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("differentiable training operators are not captured into CUDA graphs: capture the explicit forward and backward functions")
