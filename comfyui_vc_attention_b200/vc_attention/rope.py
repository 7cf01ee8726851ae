"""RMS norm of query / key heads and the position rotation, in one pass.

H3 normalises each head's query and key rows (``qk_norm_eps``) and rotates
part of the channels (MM-RoPE, 96 of 128) right before attention;
``qk_norm_rope`` does both for Q and K with one kernel launch
(``vcattn_qk_norm_rope``) and reads strided views, so the output of a fused
QKV projection needs no split copy.  ``rope_tables`` builds the cos / sin
tables, one row per token.

Forward only, like every entry point of this package: a tensor that requires
a gradient is refused while gradients are enabled.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from ._host import host_ops

__all__ = ["rope_tables", "qk_norm_rope"]


def rope_tables(positions: torch.Tensor, rot_dim: Union[int, Sequence[int]], theta: float = 10000.0, *,
                scaling: str = "none", factor: float = 1.0, original_len: Optional[int] = None,
                beta_fast: float = 32.0, beta_slow: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin tables (..., N, rot/2) fp32 of the given positions.

    positions: (N,) or (B, N) for one axis; (N, A) or (B, N, A) when
    ``rot_dim`` is a sequence of A per-axis channel counts (time, height,
    width), whose angles are laid side by side.  Channel pair i of an axis
    with r channels turns by ``position * theta**(-2 i / r)``.

    scaling: for positions beyond the trained length --
      "none";
      "linear": positions divided by ``factor``;
      "ntk":    theta multiplied by ``factor**(r / (r - 2))``;
      "yarn":   per channel pair, between no change (more than ``beta_fast``
                turns over ``original_len`` positions) and "linear" (fewer than
                ``beta_slow``), with both tables multiplied by
                ``1 + 0.1 ln(factor)``.  In between the weight is linear in
                the number of turns, which is the published method's rule.
                Code that ramps over the channel index instead (between the
                rounded indices of the two bounds) gives other tables in the
                middle channels: a checkpoint trained with such tables needs
                those, passed as cos and sin.
    """
    dims = [int(rot_dim)] if isinstance(rot_dim, int) else [int(r) for r in rot_dim]
    pos = positions if not isinstance(rot_dim, int) else positions.unsqueeze(-1)
    if pos.dim() < 2 or pos.shape[-1] != len(dims):
        raise ValueError(f"positions {tuple(positions.shape)} do not hold one value per axis of rot_dim {rot_dim}")
    if any(r <= 0 or r % 2 for r in dims):
        raise ValueError(f"rot_dim must be positive and even, got {rot_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if not factor >= 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling == "yarn" and not original_len:
        raise ValueError("yarn scaling needs original_len")
    pos = pos.to(torch.float64)
    parts, mult = [], 1.0
    for i, r in enumerate(dims):
        base = theta
        if scaling == "ntk" and r > 2:
            base = theta * factor ** (r / (r - 2))
        inv = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device=pos.device) / r)
        if scaling == "linear":
            inv = inv / factor
        elif scaling == "yarn":
            turns = original_len * inv / (2 * math.pi)
            keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
            inv = inv * keep + inv / factor * (1.0 - keep)
            mult = 1.0 + 0.1 * math.log(factor)
        parts.append(pos[..., i:i + 1] * inv)
    ang = torch.cat(parts, dim=-1)
    return (ang.cos() * mult).float().contiguous(), (ang.sin() * mult).float().contiguous()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, *, layout: str = "half", eps: float = 1e-5,
                 norm: bool = True, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-head RMS norm of q and k and the rotation by ``cos`` / ``sin``.

    q: (B, Hq, N, D), k: (B, Hk, N, D) CUDA bf16 / fp16 / fp32, any strides with
    contiguous channels (others are copied); D a multiple of 8 up to 256.
    cos, sin: (N, r/2) or (B, N, r/2) tables (``rope_tables``); the first r
    channels (r a multiple of 16) are rotated in pairs (i, i + r/2) for
    ``layout="half"`` or (2i, 2i + 1) for ``"interleaved"``, the others only
    normalised.  None: no rotation.  q_weight, k_weight: (D,) norm weights or
    None (ones); ``norm=False`` leaves the norm out (the weights still apply).
    out: a (q, k) pair of tensors to write (may be the inputs).  Arithmetic in
    fp32, rounded once.
    """
    oq, ok = (None, None) if out is None else out
    return host_ops().qk_norm_rope(q, k, cos, sin, q_weight, k_weight, layout, eps, norm, oq, ok)
