"""Exact attention over packed sequences of different lengths.

The rows VC-Attention leaves to an exact kernel -- text prompts and refiner
blocks, prompt encoders (causal, grouped heads), sequences below
``min_tokens``, single new tokens against their history -- lie one after the
other in one buffer.  ``packed_plan`` lays the batch out once (the lengths are
host numbers, checked here, so no call can read past the buffers) and
``packed_attention`` runs it for every layer.

Kernels: ``vcattn_attn_packed`` (tcgen05 for sequences of many queries,
register MMAs over the rows of a KV head's group for few).  Forward only.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native as N
from ._launch import DTYPES, on_device, out_view, refuse_grad, stream, view

__all__ = ["PackedPlan", "packed_plan", "packed_attention"]

SMS = 148

# Rows of a tile, granularity of a key range, the shortest range worth a tile of
# its own, and the tiles per SM that keep it busy: register-MMA tiles of (token,
# group head) rows, and tcgen05 tiles of tokens.
FEW = (16, 64, 256, 4)
MID = (64, 64, 256, 4)
WIDE = (256, 128, 1024, 1)
WIDE_FROM = 64   # queries of a sequence that goes to the tcgen05 kernel


@dataclass(frozen=True)
class PackedPlan:
    """Work of one batch layout, on the device (made by ``packed_plan``)."""
    heads: int
    kv_heads: int
    head_dim: int
    causal: bool
    total_q: int
    total_k: int
    tiles: Tuple[torch.Tensor, ...]   # three lists of (n, 8) int32 vcattn_packed_tile records: FEW, MID, WIDE
    joins: Tuple[torch.Tensor, ...]   # and of vcattn_packed_join records
    work: N.PackedWork                # the lists for the C ABI
    workspace_bytes: int              # partial results of one call

    @property
    def device(self) -> torch.device:
        return self.tiles[0].device


def _lengths(x, what) -> np.ndarray:
    a = np.asarray([int(v) for v in x], dtype=np.int64)
    if (a < 0).any():
        raise ValueError(f"{what} must not be negative")
    if a.sum() >= 2 ** 31:
        raise ValueError(f"{what} add up to 2^31 rows or more")
    return a


def _tiles(q0, ql, k0, kl, group, heads, causal, shape):
    """Tile and join records (int32 arrays) of the given sequences, and the
    number of partial results.  A batch that would leave SMs idle splits its
    longest key ranges."""
    rows, step, least, per_sm = shape
    per = -(-(ql * group) // rows)
    seq = np.repeat(np.arange(len(ql)), per)
    r0 = (np.arange(len(seq)) - np.repeat(np.cumsum(per) - per, per)) * rows
    lq, lk = ql[seq], kl[seq]
    last = np.minimum((r0 + rows - 1) // group, lq - 1)
    ke = np.clip(last + 1 + lk - lq, 0, lk) if causal else lk.copy()
    pieces = np.ones(len(seq), dtype=np.int64)
    work = int(ke.sum()) * heads
    if len(seq) * heads < per_sm * SMS and work:
        pieces = np.maximum(1, -(-ke // max(least, -(-work // (per_sm * SMS)))))
    span = -(-(-(-ke // pieces)) // step) * step             # keys per piece
    pieces = np.maximum(1, -(-ke // np.maximum(span, 1)))
    row = np.repeat(np.arange(len(seq)), pieces)
    piece = np.arange(len(row)) - np.repeat(np.cumsum(pieces) - pieces, pieces)
    kb = piece * span[row]
    split = pieces[row] > 1
    slot = np.where(split, np.cumsum(split) - 1, -1)
    tiles = np.stack([q0[seq][row], lq[row], k0[seq][row], lk[row], r0[row], kb,
                      np.minimum(kb + span[row], ke[row]), slot], axis=1).astype(np.int32)
    tiles = np.ascontiguousarray(tiles[np.argsort(-(tiles[:, 6] - tiles[:, 5]), kind="stable")])   # longest first
    js = np.nonzero(pieces > 1)[0]
    joins = np.zeros((len(js), 8), dtype=np.int32)
    joins[:, 0], joins[:, 1], joins[:, 2] = q0[seq][js], lq[js], r0[js]
    joins[:, 3], joins[:, 4] = np.cumsum(pieces[js]) - pieces[js], pieces[js]
    return tiles, joins, int(split.sum())


def packed_plan(q_lens: Sequence[int], k_lens: Optional[Sequence[int]] = None, *, heads: int,
                kv_heads: Optional[int] = None, head_dim: int, causal: bool = False,
                device: Optional[torch.device] = None) -> PackedPlan:
    """Lay out a batch: sequence i has q_lens[i] queries and k_lens[i] keys
    (default: as many), the rows of sequence i + 1 following those of i.

    causal: query t of lq sees keys up to t + lk - lq (the last query sees
    every key, as when lq new tokens follow a history); a query before the
    first key sees none and its output is 0.  heads must be a multiple of
    kv_heads (default: heads); head_dim is 64 or 128.
    """
    kv_heads = heads if kv_heads is None else kv_heads
    ql = _lengths(q_lens, "q_lens")
    kl = ql if k_lens is None else _lengths(k_lens, "k_lens")
    if len(ql) != len(kl):
        raise ValueError(f"{len(ql)} query lengths and {len(kl)} key lengths")
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise ValueError(f"heads ({heads}) must be a positive multiple of kv_heads ({kv_heads})")
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
    g = heads // kv_heads
    if (ql * g >= 2 ** 31).any():
        raise ValueError("a sequence has 2^31 rows or more")
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    q0, k0 = np.cumsum(ql) - ql, np.cumsum(kl) - kl
    wide, few = ql >= WIDE_FROM, ql * g <= FEW[0]
    lists = ((few & ~wide, g, kv_heads, FEW), (~few & ~wide, g, kv_heads, MID), (wide, 1, heads, WIDE))
    tiles, joins, slots, need = [], [], [], 0
    for pick, group, hs, shape in lists:
        t, j, n = _tiles(q0[pick], ql[pick], k0[pick], kl[pick], group, hs, causal, shape)
        tiles.append(torch.from_numpy(t).to(dev))
        joins.append(torch.from_numpy(j).to(dev))
        slots.append(n)
        need += n * hs * shape[0] * (head_dim + 2) * 4
    work = N.PackedWork(tuple(t.data_ptr() for t in tiles), tuple(j.data_ptr() for j in joins),
                        tuple(t.shape[0] for t in tiles), tuple(j.shape[0] for j in joins), tuple(slots))
    return PackedPlan(heads, kv_heads, head_dim, bool(causal), int(ql.sum()), int(kl.sum()), tuple(tiles), tuple(joins),
                      work, need)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T + mask) v for every sequence of ``plan``.

    q: (1, heads, total_q, D), k, v: (1, kv_heads, total_k, D) CUDA bf16 or
    fp16 views (channels contiguous; others are copied).  scale: positive,
    default D ** -0.5.  Returns (1, heads, total_q, D) in q's token layout, or
    writes ``out``.  Scores, statistics and sums are fp32; P is rounded to q's
    type for the second product.
    """
    if torch.is_grad_enabled():
        refuse_grad("packed_attention", q, k, v)
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise RuntimeError("packed_attention needs CUDA tensors (this build has no CPU path)")
    d = plan.head_dim
    want_q, want_k = (1, plan.heads, plan.total_q, d), (1, plan.kv_heads, plan.total_k, d)
    if q.shape != want_q or k.shape != want_k or v.shape != want_k:
        raise ValueError(f"the plan needs q {want_q} and k, v {want_k}, got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    dtype, dev = q.dtype, q.device
    if dtype not in (torch.bfloat16, torch.float16) or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"q, k, v must share bfloat16 or float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if not dev == k.device == v.device == plan.device:
        raise ValueError("q, k, v and the plan must be on one device")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    ov, out = out_view(out, q, "out")
    (qv, q), (kv, k), (vv, v) = view(q), view(k), view(v)   # (what a view points into lives until the launch)
    need, ws = plan.workspace_bytes, None
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with on_device(dev):
        N.check("vcattn_attn_packed", N.lib().vcattn_attn_packed(
            qv, kv, vv, DTYPES[dtype], plan.heads, plan.kv_heads, plan.total_q, plan.total_k, d, plan.work, plan.causal,
            scale, ov, None if ws is None else ws.data_ptr(), need, stream(dev)))
    return out
