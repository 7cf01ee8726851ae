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

from . import _native as N
from ._launch import DTYPES, on_device, out_view, refuse_grad, stream, view

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
                ``1 + 0.1 ln(factor)``.
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


def _vector(w: torch.Tensor, d: int, device: torch.device, what: str) -> torch.Tensor:
    """A (D,) weight as the kernel reads it: fp32, contiguous, 16-byte aligned."""
    if w.shape != (d,):
        raise ValueError(f"{what} must be ({d},), got {tuple(w.shape)}")
    if w.device != device:
        raise ValueError(f"{what} must be on {device}, got {w.device}")
    if w.dtype != torch.float32:
        w = w.to(torch.float32)
    return w if w.stride(0) == 1 and w.data_ptr() & 15 == 0 else w.clone(memory_format=torch.contiguous_format)


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
    if torch.is_grad_enabled():
        refuse_grad("qk_norm_rope", q, k, cos, sin, q_weight, k_weight)
    if not (q.is_cuda and k.is_cuda):
        raise RuntimeError("qk_norm_rope needs CUDA tensors (this build has no CPU path)")
    qs, ks, dev, dtype = q.shape, k.shape, q.device, q.dtype
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError(f"q and k must be (B, Hq, N, D) and (B, Hk, N, D), got {tuple(qs)}, {tuple(ks)}")
    b, hq, n, d = qs
    if ks != (b, ks[1], n, d):
        raise ValueError(f"q and k must be (B, Hq, N, D) and (B, Hk, N, D), got {tuple(qs)}, {tuple(ks)}")
    if k.dtype != dtype or k.device != dev:
        raise ValueError("q and k must share a dtype and a device")
    dt = DTYPES.get(dtype)
    if dt is None:
        raise TypeError(f"unsupported dtype {dtype}")
    if d & 7 or not 8 <= d <= 256:
        raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {d}")
    if layout == "half":
        flags = N.ROPE_NORM if norm else 0
    elif layout == "interleaved":
        flags = N.ROPE_INTERLEAVED | (N.ROPE_NORM if norm else 0)
    else:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    rot = tsb = tsn = 0
    cp = sp = None
    if cos is not None and sin is not None:
        cs = cos.shape
        if cs != sin.shape or len(cs) not in (2, 3) or cs[-2] != n or (len(cs) == 3 and cs[0] not in (1, b)):
            raise ValueError(f"cos and sin must be ({n}, r/2) or ({b}, {n}, r/2), got {tuple(cs)}, {tuple(sin.shape)}")
        if cos.device != dev or sin.device != dev:
            raise ValueError(f"cos and sin must be on {dev}")
        rot = 2 * cs[-1]
        if rot & 15 or rot > d:
            raise ValueError(f"the rotated channels must be a multiple of 16 up to {d}, got {rot}")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            cos, sin = cos.to(torch.float32), sin.to(torch.float32)
        st = cos.stride()
        if st != sin.stride() or st[-1] != 1 or (st[0] | st[-2]) & 3 or (cos.data_ptr() | sin.data_ptr()) & 15:
            cos, sin = (x.clone(memory_format=torch.contiguous_format) for x in (cos, sin))
            st = cos.stride()
        tsn = st[-2]
        tsb = st[0] if len(st) == 3 and cs[0] > 1 else 0
        cp, sp = cos.data_ptr(), sin.data_ptr()
    elif cos is not None or sin is not None:
        raise ValueError("cos and sin are given together")
    qw = kw = None
    if q_weight is not None:
        q_weight = _vector(q_weight, d, dev, "q_weight")
        qw = q_weight.data_ptr()
    if k_weight is not None:
        k_weight = _vector(k_weight, d, dev, "k_weight")
        kw = k_weight.data_ptr()
    oq, ok = (None, None) if out is None else out
    (ov, oq), (pv, ok) = out_view(oq, q, "out[0]"), out_view(ok, k, "out[1]")
    (qv, q), (kv, k) = view(q), view(k)   # (what a view points into lives until the launch)
    with on_device(dev):
        N.check("vcattn_qk_norm_rope", N.lib().vcattn_qk_norm_rope(
            qv, kv, dt, b, hq, ks[1], n, d, qw, kw, cp, sp, tsb, tsn, rot, flags, eps, ov, pv, stream(dev)))
    return oq, ok
