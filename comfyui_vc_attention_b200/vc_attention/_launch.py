"""What the host sides of the block operators share: strided views for the C
ABI, output buffers, the device guard and the refusal of gradients."""

from __future__ import annotations

from contextlib import nullcontext
from typing import Optional, Tuple

import torch

from . import _native as N

_SAME_DEVICE = nullcontext()


def refuse_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """The operators have no backward pass: say so instead of cutting the graph."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")


def on_device(device: torch.device):
    """Context in which ``device`` is current (nothing to do when it already is)."""
    return _SAME_DEVICE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def rows_aligned(x: torch.Tensor) -> bool:
    """(B, H, N, D) with contiguous channels and every row on a 16-byte boundary."""
    sb, sh, sn, sd = x.stride()
    return sd == 1 and (x.data_ptr() | sb * x.element_size() | sh * x.element_size() | sn * x.element_size()) & 15 == 0


def view(x: torch.Tensor) -> Tuple[N.BHND, torch.Tensor]:
    """vcattn_bhnd of x and the tensor it points into (a copy if the rows are
    not aligned, or are the same memory as those of a broadcast view)."""
    if not rows_aligned(x) or (0 in x.stride() and x.numel() > x.shape[-1]):
        x = x.clone(memory_format=torch.contiguous_format)
    sb, sh, sn, _ = x.stride()
    return N.BHND(x.data_ptr(), sb, sh, sn), x


def empty_like_rows(x: torch.Tensor) -> torch.Tensor:
    """Output buffer in the token layout of a (B, H, N, D) input: token-major
    rows (the ComfyUI (B, N, H*D) path) stay token-major."""
    b, h, n, d = x.shape
    if x.stride(1) < x.stride(2):
        return torch.empty((b, n, h, d), dtype=x.dtype, device=x.device).transpose(1, 2)
    return torch.empty((b, h, n, d), dtype=x.dtype, device=x.device)


def out_rows(out: Optional[torch.Tensor], x: torch.Tensor, what: str) -> torch.Tensor:
    """``out`` checked against its input, or a new buffer."""
    if out is None:
        return empty_like_rows(x)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{what} must match its input: {tuple(x.shape)} {x.dtype} on {x.device}")
    if out.numel() and (not rows_aligned(out) or any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape))):
        raise ValueError(f"{what} must have contiguous channels and 16-byte aligned rows of their own")
    return out
