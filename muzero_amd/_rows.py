"""What the row operators (policy scores, 8-bit codes, products and checkpoints) share on the host side: element
types, two-dimensional views of their arguments, the stream and device a call belongs to."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from muzero_amd import _hip

TYPE = {torch.float32: _hip.TYPE_F32, torch.bfloat16: _hip.TYPE_BF16, torch.float16: _hip.TYPE_F16}
MAX_ROWS, MAX_COLUMNS = (1 << 31) - 1, 1 << 30
_NULL = contextlib.nullcontext()


def check_tensor(t: torch.Tensor, what: str, forward_mode: bool = False) -> None:
    """A float32 / bfloat16 / float16 tensor on the GPU, without a forward-mode tangent unless the caller sees to it, or an
    error that says which."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, not {type(t).__name__}")
    if t.dtype not in TYPE:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    if not forward_mode:
        refuse_tangent(t, what)
    check_on_gpu(t, what)


def refuse_tangent(t: torch.Tensor, what: str) -> None:
    """The kernels have no forward-mode derivative, and a result without a tangent would read as one that does not depend
    on t.  (torch.no_grad() does not switch forward mode off.)"""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:  # no call where no level is open
        raise NotImplementedError(f"{what} carries a forward-mode tangent, for which there is no derivative here")


def check_on_gpu(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise _hip.HipError(f"{what} must be on the GPU (there is no CPU fallback for the kernels)")


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, columns] with adjacent columns and rows that do not overlap: a view where its strides allow one, else
    a copy."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.dim() != 2:
        cols = t.shape[-1]
        t = t.reshape(-1, cols) if cols else t.reshape(t.shape[:-1].numel(), 0)
    (rows, cols), (step, one) = t.shape, t.stride()
    if (cols > 1 and one != 1) or (rows > 1 and step < cols):
        t = t.contiguous()
    if rows > MAX_ROWS or cols > MAX_COLUMNS:
        raise ValueError(f"{rows} rows of {cols} values are more than a call takes ({MAX_ROWS} of {MAX_COLUMNS})")
    return t


def in_memory(t: torch.Tensor) -> torch.Tensor:
    """t with adjacent values as its memory holds them: the minus sign of a view (the imaginary part of a conjugate, say)
    is not in memory, and contiguous() leaves it out where the strides fit."""
    return (t.resolve_neg() if t.is_neg() else t).contiguous()


def row_stride(t: torch.Tensor) -> int:
    """Elements from one row of rows_of's result to the next (a single row may carry any stride)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def on_device(t: torch.Tensor):
    """Context in which t's device is the current one."""
    return _NULL if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)


def stream_of(t: torch.Tensor) -> int:
    """The current stream of t's device, as the handle itself: torch.cuda.current_stream(...).cuda_stream costs 2 us a
    call, half of a small launch."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def workspace(nbytes: int, t: torch.Tensor) -> torch.Tensor | None:
    """Scratch memory of one call, from torch's allocator: it belongs to the stream the call runs on."""
    if nbytes < 0:
        raise _hip.HipError("bad workspace size")
    return torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes > 0 else None
