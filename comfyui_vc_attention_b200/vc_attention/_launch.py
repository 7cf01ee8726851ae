"""What the host sides of the block operators share: strided views for the C
ABI, output buffers, the device guard and the refusal of gradients."""

from __future__ import annotations

from contextlib import nullcontext
from typing import Optional, Tuple

import torch

from . import _native as N

DTYPES = {torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16, torch.float32: N.DTYPE_F32}

_SAME_DEVICE = nullcontext()
# The current device and raw stream without building Python objects for them
# (a call's host time is what a small launch costs); the public calls where a
# torch build lacks these.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def refuse_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """The operators have no backward pass: say so instead of cutting the graph."""
    for t in tensors:
        if t is not None and t.requires_grad:
            raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")


def on_device(device: torch.device):
    """Context in which ``device`` is current (nothing to do when it already is)."""
    return _SAME_DEVICE if _current_device() == device.index else torch.cuda.device(device)


def stream(device: torch.device) -> int:
    """The current stream of ``device``."""
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def view(x: torch.Tensor) -> Tuple[N.BHND, torch.Tensor]:
    """vcattn_bhnd of a (B, H, N, D) tensor and the tensor it points into: a
    copy if the channels are not contiguous, a row is not on a 16-byte boundary
    or rows are the same memory (a broadcast view)."""
    sb, sh, sn, sd = x.stride()
    p = x.data_ptr()
    if sd != 1 or (p | (sb | sh | sn) * x.element_size()) & 15 or not (sb and sh and sn):
        x = x.clone(memory_format=torch.contiguous_format)
        sb, sh, sn, _ = x.stride()
        p = x.data_ptr()
    return N.BHND(p, sb, sh, sn), x


def out_view(out: Optional[torch.Tensor], x: torch.Tensor, what: str) -> Tuple[N.BHND, torch.Tensor]:
    """``out`` checked against its input, or a new buffer in the token layout of
    the input: token-major rows (the ComfyUI (B, N, H*D) path) stay so."""
    if out is None:
        out = torch.empty_like(x)   # (dense, dimensions in x's order)
        sb, sh, sn, sd = out.stride()
        if sd != 1:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            sb, sh, sn, _ = out.stride()
        return N.BHND(out.data_ptr(), sb, sh, sn), out
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{what} must match its input: {tuple(x.shape)} {x.dtype} on {x.device}")
    sb, sh, sn, sd = out.stride()
    if out.numel() and (sd != 1 or (out.data_ptr() | (sb | sh | sn) * out.element_size()) & 15
                        or any(s == 0 and m > 1 for s, m in zip(out.stride(), out.shape))):
        raise ValueError(f"{what} must have contiguous channels and 16-byte aligned rows of their own")
    return N.BHND(out.data_ptr(), sb, sh, sn), out
