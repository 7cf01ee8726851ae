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

from ._host import host_ops

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
    codes, scale = host_ops().quantize_blocks(x, rows)
    return Fp8Blocks(codes, scale, rows)


def matmul_blocks(a: Fp8Blocks, b: Fp8Blocks, bias: Optional[torch.Tensor] = None,
                  dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ b.T (+ bias): (M, K) x (N, K) -> (M, N) in ``dtype``.

    a has rows=1 (activations), b rows=128 (weights); each product of 128
    columns is scaled by both blocks' scales and added in fp32, and the result
    is rounded once.  bias: (N,) or None.  out: (M, N) of ``dtype`` with
    contiguous columns, or None.
    """
    return host_ops().matmul_blocks(a.codes, a.scale, a.rows, b.codes, b.scale, b.rows, bias, dtype, out)


def linear_blocks(x: torch.Tensor, weight: Fp8Blocks, bias: Optional[torch.Tensor] = None,
                  dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x (..., K) times a quantised (N, K) weight: (..., N) in ``dtype`` (x's by default)."""
    y = matmul_blocks(quantize_blocks(x), weight, bias, dtype or x.dtype)
    return y.view(*x.shape[:-1], y.shape[-1])
