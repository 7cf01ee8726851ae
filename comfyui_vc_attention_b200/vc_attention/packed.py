"""Exact attention over packed sequences of different lengths.

The rows VC-Attention leaves to an exact kernel -- text prompts and refiner
blocks, prompt encoders (causal, grouped heads), sequences below
``min_tokens``, single new tokens against their history -- lie one after the
other in one buffer.  ``packed_plan`` lays the batch out once (the lengths are
host numbers, checked here, so no call can read past the buffers) and
``packed_attention`` runs it for every layer.

Kernels: ``vcattn_attn_packed`` (tcgen05 for sequences of many queries,
register MMAs over the rows of a KV head's group for few).  Forward only.

A plan may be used on any stream and dropped while its calls still run: the
records that the kernels read stay until then, and as long as a captured graph
needs them.
"""

from __future__ import annotations

import ctypes
import math
import operator
from dataclasses import dataclass
from typing import NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _native as N
from ._host import host_ops

__all__ = ["PackedPlan", "packed_plan", "packed_attention"]

SMS = 148


class _Shape(NamedTuple):
    """One of the three kinds of tiles: rows per tile, granularity of a key
    range, CTAs resident on the SMs, and what a tile, a part of a split tile
    and a join cost beside their keys, in keys (for the choice of a split)."""
    rows: int
    step: int
    slots: int
    tile_cost: int
    part_cost: int
    join_cost: int


# Register-MMA tiles of (token, group head) rows, and tcgen05 tiles of tokens.
FEW = _Shape(16, 64, 2 * SMS, 0, 0, 0)
MID = _Shape(64, 64, 3 * SMS, 128, 100, 160)
WIDE = _Shape(256, 128, SMS, 320, 450, 640)
# A tcgen05 tile takes about 0.55 of a 64-row register-MMA tile over the same
# keys, but covers one query head where that covers a group's.  8 sequences of
# 4096 keys, 32 / 8 heads, in us, tcgen05 / register MMAs: 24 queries 107 / 98,
# 32 107 / 100, 48 112 / 145, 128 114 / 367; 56 / 56 heads, 1024 keys: 16
# queries (16-row tiles) 37 / 30, 24 38 / 58.
WIDE_TILE = 0.55


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
    call: object                      # the same for the host extension, which keeps the records while a call reads them

    @property
    def device(self) -> torch.device:
        return self.tiles[0].device


def _lengths(x, what) -> np.ndarray:
    try:
        n = [operator.index(v) for v in x]
    except TypeError as e:
        raise TypeError(f"{what} must be whole numbers") from e
    if any(v < 0 for v in n):
        raise ValueError(f"{what} must not be negative")
    if sum(n) >= 2 ** 31:   # (in Python's numbers: in 64 bits the sum may wrap)
        raise ValueError(f"{what} add up to 2^31 rows or more")
    return np.asarray(n, dtype=np.int64)


def _pieces(ke: np.ndarray, heads: int, shape: _Shape):
    """Key ranges per tile and their length, for tiles of ``ke`` keys on each of
    ``heads`` heads."""
    def spans(share):
        n = np.maximum(1, -(-ke // share))
        span = np.maximum(shape.step, -(-(-(-ke // n)) // shape.step) * shape.step)
        return np.maximum(1, -(-ke // span)), span

    total, longest = int(ke.sum()) * heads, max(1, int(ke.max(initial=0)))
    if shape is FEW:
        # Bound by the K/V bytes, which one CTA per SM nearly draws: tiles are
        # split only where one holds more than an SM's share (12 sequences of 1
        # to 8192 keys: 45 us unsplit at two CTAs' share, 38 us; 64 of 2048:
        # 91 us whole, 103 in halves).
        return spans(longest if longest <= total / SMS else max(4 * shape.step, math.ceil(total / shape.slots)))
    # Bound by the tensor cores: splitting evens out the CTAs and costs partial
    # results and a join.  Of a few splits, the one whose longest run of CTAs on
    # a slot is estimated shortest (longest first: no shorter than the longest
    # tile, the mean, and the two tiles that meet where the slots run out).
    best = None
    for c in (0.0, 0.75, 1.0, 1.5, 2.0, 3.0):
        share = max(4 * shape.step, math.ceil(total / (shape.slots * c))) if c else longest
        if c and share >= longest:
            continue
        n, span = spans(share)
        size = np.repeat(np.minimum(span, ke) + np.where(n > 1, shape.part_cost, 0) + shape.tile_cost, n)
        size = np.sort(size)[::-1]
        cost = max(int(size[0]), int(size.sum()) * heads / shape.slots)
        at = shape.slots // heads
        if 0 < at < len(size):
            cost = max(cost, int(size[at - 1]) + int(size[at]))
        cost += shape.join_cost if (n > 1).any() else 0
        if best is None or cost < best[0]:
            best = (cost, n, span)
    return best[1], best[2]


def _tiles(q0, ql, k0, kl, group, heads, causal, shape: _Shape):
    """Tile and join records (int32 arrays) of the given sequences, and the
    number of partial results."""
    none = np.zeros((0, 8), dtype=np.int32)
    if not ql.any():
        return none, none, 0
    per = -(-(ql * group) // shape.rows)
    seq = np.repeat(np.arange(len(ql)), per)
    r0 = (np.arange(len(seq)) - np.repeat(np.cumsum(per) - per, per)) * shape.rows
    lq, lk = ql[seq], kl[seq]
    last = np.minimum((r0 + shape.rows - 1) // group, lq - 1)
    ke = np.clip(last + 1 + lk - lq, 0, lk) if causal else lk
    pieces, span = _pieces(ke, heads, shape)
    row = np.repeat(np.arange(len(seq)), pieces)
    piece = np.arange(len(row)) - np.repeat(np.cumsum(pieces) - pieces, pieces)
    kb = piece * span[row]
    split = pieces[row] > 1
    slot = np.where(split, np.cumsum(split) - 1, -1)
    tiles = np.stack([q0[seq][row], lq[row], k0[seq][row], lk[row], r0[row], kb,
                      np.minimum(kb + span[row], ke[row]), slot], axis=1).astype(np.int32)
    tiles = tiles[np.argsort(tiles[:, 5] - tiles[:, 6], kind="stable")]   # longest first
    js = np.nonzero(pieces > 1)[0]
    if not len(js):
        return tiles, none, 0
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
    few = ql * g <= FEW.rows
    wide = ~few & (WIDE_TILE * g < -(-ql * g // MID.rows))
    lists = ((few, g, kv_heads, FEW), (~few & ~wide, g, kv_heads, MID), (wide, 1, heads, WIDE))
    made = [_tiles(q0[pick], ql[pick], k0[pick], kl[pick], group, hs, causal, shape)
            for pick, group, hs, shape in lists]
    need = sum(m[2] * hs * shape.rows * (head_dim + 2) * 4 for m, (_, _, hs, shape) in zip(made, lists))
    # one upload for all records
    host = np.concatenate([m[i] for i in (0, 1) for m in made])
    records = torch.from_numpy(host).to(dev)
    recs = records.split([len(m[i]) for i in (0, 1) for m in made])
    work = N.PackedWork(tuple(r.data_ptr() for r in recs[:3]), tuple(r.data_ptr() for r in recs[3:]),
                        tuple(len(r) for r in recs[:3]), tuple(len(r) for r in recs[3:]), tuple(m[2] for m in made))
    tq, tk = int(ql.sum()), int(kl.sum())
    call = host_ops().packed_call(heads, kv_heads, tq, tk, head_dim, bool(causal), ctypes.addressof(work), need, records)
    return PackedPlan(heads, kv_heads, head_dim, bool(causal), tq, tk, recs[:3], recs[3:], work, need, call)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PackedPlan,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T + mask) v for every sequence of ``plan``.

    q: (1, heads, total_q, D), k, v: (1, kv_heads, total_k, D) CUDA bf16 or
    fp16 views (channels contiguous; others are copied), the sequences' rows one
    after the other.  scale: positive, default D ** -0.5.  Returns (1, heads,
    total_q, D) in q's token layout, or writes ``out``, which may be q but not
    overlap k or v.  Scores, statistics and sums are fp32; P is rounded to q's
    type for the second product (in fp16 to 2^-11 of itself or 2^-36 of the
    row's largest).
    """
    return host_ops().packed_attention(q, k, v, plan.call, scale, out)
