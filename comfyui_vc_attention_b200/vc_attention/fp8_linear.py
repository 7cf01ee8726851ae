"""8-bit linear layers: E4M3 codes with one scale for each block of 128.

Activations are quantised per (row, 128 columns), weights per (128 x 128), and
the product applies both scales to each block's partial sum in fp32::

    w = quantize_blocks(weight, rows=128)          # once
    y = linear_blocks(x, w, bias)                  # quantize_blocks(x) + matmul_blocks

Kernels: ``vcattn_quantize_blocks`` and ``vcattn_matmul_blocks`` (tcgen05).
Forward only.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as N
from ._launch import DTYPES, on_device, refuse_grad, stream

__all__ = ["Fp8Blocks", "quantize_blocks", "matmul_blocks", "linear_blocks"]

BLOCK = 128


class Fp8Blocks(NamedTuple):
    """A quantised (M, K) matrix: value = codes * scale of its block."""
    codes: torch.Tensor   # (M, K) float8_e4m3fn, row pitch a multiple of 16
    scale: torch.Tensor   # (ceil(M / rows), ceil(K / 128)) fp32
    rows: int             # 1 or 128 rows per block


def quantize_blocks(x: torch.Tensor, rows: int = 1) -> Fp8Blocks:
    """E4M3 codes and scales of x, (M, K) or (..., K) with the leading
    dimensions flattened; CUDA bf16 / fp16 / fp32.

    rows=1: a scale per row and 128 columns (activations); rows=128: per
    128 x 128 block (weights).  scale = max(max |x|, 1e-30) / 448, codes =
    E4M3(x / scale), round to nearest even.  The scales are stored with rows
    side by side (the order the product reads them in).
    """
    if x.requires_grad and torch.is_grad_enabled():
        refuse_grad("quantize_blocks", x)
    if not x.is_cuda:
        raise RuntimeError("quantize_blocks needs a CUDA tensor (this build has no CPU path)")
    if rows not in (1, BLOCK):
        raise ValueError(f"rows must be 1 or {BLOCK}, got {rows}")
    dt = DTYPES.get(x.dtype)
    if dt is None:
        raise TypeError(f"unsupported dtype {x.dtype}")
    xs = x.shape
    if len(xs) < 1 or xs[-1] == 0:
        raise ValueError(f"x must be (M, K) with K > 0, got {tuple(xs)}")
    k = xs[-1]
    x2 = x if len(xs) == 2 else x.reshape(-1, k)
    m = x2.shape[0]
    ldx, sk = x2.stride()
    if (sk != 1 and k > 1) or (m > 1 and ldx < k):
        x2 = x2.clone(memory_format=torch.contiguous_format)
        ldx = k
    dev = x.device
    ldc = -(-k // 16) * 16
    # (empty_strided: half the host time of empty, and the padded pitch in one call)
    codes = torch.empty_strided((m, k), (ldc, 1), dtype=torch.float8_e4m3fn, device=dev)
    mb = m if rows == 1 else -(-m // rows)
    scale = torch.empty_strided((mb, -(-k // BLOCK)), (1, mb), dtype=torch.float32, device=dev)
    with on_device(dev):
        N.check("vcattn_quantize_blocks", N.lib().vcattn_quantize_blocks(
            x2.data_ptr(), dt, m, k, max(ldx, k), rows, codes.data_ptr(), ldc, scale.data_ptr(), 1, mb, stream(dev)))
    return Fp8Blocks(codes, scale, rows)


def _code_rows(b: Fp8Blocks, name: str, rows: int):
    """(codes, row pitch) of a checked operand as the TMA reads them: 16-byte rows, copied if need be."""
    c, s = b.codes, b.scale
    if not (c.is_cuda and s.is_cuda) or c.device != s.device:
        raise RuntimeError(f"matmul_blocks needs CUDA tensors on one device ({name})")
    if b.rows != rows:
        raise ValueError(f"{name} must have one scale per {rows} row(s) and {BLOCK} columns, got rows={b.rows}")
    if c.dtype != torch.float8_e4m3fn or c.dim() != 2 or c.shape[1] == 0:
        raise ValueError(f"{name}.codes must be (rows, K) float8_e4m3fn, got {tuple(c.shape)} {c.dtype}")
    m, k = c.shape
    if s.dtype != torch.float32 or s.shape != (-(-m // rows), -(-k // BLOCK)):
        raise ValueError(f"{name}.scale must be {(-(-m // rows), -(-k // BLOCK))} float32, got {tuple(s.shape)} {s.dtype}")
    ld, sk = c.stride()
    if m <= 1:
        ld = -(-k // 16) * 16   # (the pitch of a single row is never used)
    if (sk == 1 or k == 1) and (c.data_ptr() | ld) & 15 == 0 and ld >= k:
        return c, ld
    ld = -(-k // 16) * 16
    t = torch.empty((m, ld), dtype=c.dtype, device=c.device)
    t[:, :k].copy_(c)
    return t, ld


def matmul_blocks(a: Fp8Blocks, b: Fp8Blocks, bias: Optional[torch.Tensor] = None,
                  dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ b.T (+ bias): (M, K) x (N, K) -> (M, N) in ``dtype``.

    a has rows=1 (activations), b rows=128 (weights); each product of 128
    columns is scaled by both blocks' scales and added in fp32, and the result
    is rounded once.  bias: (N,) or None.  out: (M, N) of ``dtype`` with
    contiguous columns, or None.
    """
    if torch.is_grad_enabled():
        refuse_grad("matmul_blocks", a.scale, b.scale, bias)
    ac, lda = _code_rows(a, "a", 1)
    bc, ldb = _code_rows(b, "b", BLOCK)
    m, k = a.codes.shape
    n, kb = b.codes.shape
    dev = ac.device
    if kb != k or bc.device != dev:
        raise ValueError(f"a and b must share K and a device, got {tuple(a.codes.shape)} on {dev}, "
                         f"{tuple(b.codes.shape)} on {bc.device}")
    bp = None
    if bias is not None:
        if bias.shape != (n,) or bias.device != dev:
            raise ValueError(f"bias must be ({n},) on {dev}, got {tuple(bias.shape)} on {bias.device}")
        if bias.dtype != torch.float32 or bias.stride(0) != 1:
            bias = bias.to(torch.float32).contiguous()
        bp = bias.data_ptr()
    odt = DTYPES.get(dtype)
    if odt is None:
        raise TypeError(f"unsupported dtype {dtype}")
    if out is None:
        ldo = max(n, 1)
        out = torch.empty_strided((m, n), (ldo, 1), dtype=dtype, device=dev)
    else:
        if out.shape != (m, n) or out.dtype != dtype or out.device != dev or (n > 1 and out.stride(1) != 1) or \
                (m > 1 and out.stride(0) < n):
            raise ValueError(f"out must be ({m}, {n}) {dtype} on {dev} with contiguous columns")
        ldo = out.stride(0) if m > 1 else max(n, 1)
    (sam, sak), (sbn, sbk) = a.scale.stride(), b.scale.stride()
    lib, wp = N.lib(), None
    with on_device(dev):
        need = lib.vcattn_matmul_blocks_workspace_bytes(m, n, k) if m > 32 else 0   # (few rows never need one)
        if need:
            ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=dev)
            wp = ws.data_ptr()
        N.check("vcattn_matmul_blocks", lib.vcattn_matmul_blocks(
            ac.data_ptr(), lda, a.scale.data_ptr(), sam, sak, bc.data_ptr(), ldb, b.scale.data_ptr(), sbn, sbk, m, n, k,
            bp, out.data_ptr(), odt, ldo, wp, need, stream(dev)))
    return out


def linear_blocks(x: torch.Tensor, weight: Fp8Blocks, bias: Optional[torch.Tensor] = None,
                  dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (..., K) times a quantised (N, K) weight: (..., N) in ``dtype`` (x's by default)."""
    y = matmul_blocks(quantize_blocks(x), weight, bias, dtype or x.dtype)
    return y.view(*x.shape[:-1], y.shape[-1])
