"""Host side of the block operators (no GPU): rotation tables, the layout of a
packed batch, and the argument checks of the C entry points."""

import ctypes
import math

import numpy as np
import pytest
import torch

from comfyui_vc_attention_b200.vc_attention import (packed_attention, packed_plan, qk_norm_rope, quantize_blocks,
                                                    rope_tables)
from comfyui_vc_attention_b200.vc_attention import _native as N


def test_rope_tables_one_axis():
    pos = torch.tensor([0, 1, 7, 100000])
    cos, sin = rope_tables(pos, 64, theta=10000.0)
    assert cos.shape == (4, 32) and cos.dtype == torch.float32
    for n, p in enumerate(pos.tolist()):
        for i in (0, 5, 31):
            a = p * 10000.0 ** (-2 * i / 64)
            assert abs(cos[n, i].item() - math.cos(a)) < 1e-7 and abs(sin[n, i].item() - math.sin(a)) < 1e-7


def test_rope_tables_axes_lie_side_by_side():
    pos = torch.tensor([[[3, 1, 2], [0, 5, 4]]])
    cos, _ = rope_tables(pos, (32, 32, 32))
    assert cos.shape == (1, 2, 48)
    for axis in range(3):
        want, _ = rope_tables(pos[..., axis], 32)
        assert torch.equal(cos[..., 16 * axis:16 * axis + 16], want)


def test_rope_tables_scaling():
    pos = torch.arange(50)
    base = rope_tables(pos, 64)
    lin = rope_tables(pos * 4, 64, scaling="linear", factor=4.0)
    assert torch.allclose(lin[0], base[0], atol=1e-7)
    ntk = rope_tables(pos, 64, scaling="ntk", factor=4.0)
    assert torch.equal(ntk[0][:, 0], base[0][:, 0])                       # fastest pair unchanged
    slow = 4.0 ** (64 / 62) * 10000.0
    assert abs(ntk[0][49, 31].item() - math.cos(49 * slow ** (-62 / 64))) < 1e-7
    y = rope_tables(pos, 64, scaling="yarn", factor=8.0, original_len=4096)
    m = 1 + 0.1 * math.log(8.0)
    assert abs(y[0][3, 0].item() - m * math.cos(3.0)) < 1e-6              # 652 turns: unchanged
    inv = 10000.0 ** (-62 / 64)                                           # 0.09 turns: linear
    assert abs(y[1][3, 31].item() - m * math.sin(3 * inv / 8)) < 1e-6


def test_rope_tables_refusals():
    pos = torch.arange(4)
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=(16, 16)), dict(rot_dim=16, scaling="other"),
                dict(rot_dim=16, scaling="linear", factor=0.5), dict(rot_dim=16, scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            rope_tables(pos, **bad)


def _covered(tiles, joins, g, size, step, ql, kl):
    """Times each (row, key) pair of each sequence is visited, and the rows written."""
    seen = [np.zeros((a * g, b), dtype=int) for a, b in zip(ql, kl)]
    rows = [np.zeros(a * g, dtype=int) for a in ql]
    q0 = np.cumsum(ql) - ql
    joined = {}
    for j in joins.numpy():
        assert j[4] >= 2
        for s in range(j[3], j[3] + j[4]):
            assert s not in joined
            joined[s] = (j[0], j[2])
    used = set()
    for t in tiles.numpy():
        i = [x for x in range(len(ql)) if q0[x] == t[0] and ql[x] == t[1] and t[1] > 0][0]
        r = slice(t[4], min(t[4] + size, ql[i] * g))
        assert r.start < r.stop and 0 <= t[5] <= max(t[5], t[6]) <= kl[i] and t[5] % step == 0
        seen[i][r, t[5]:t[6]] += 1
        if t[7] < 0:
            rows[i][r] += 1
        else:
            assert joined[t[7]] == (t[0], t[4]) and t[7] not in used
            used.add(t[7])
    assert used == set(joined)
    for j in joins.numpy():
        i = [x for x in range(len(ql)) if q0[x] == j[0] and ql[x] == j[1] and ql[x] > 0][0]
        rows[i][j[2]:min(j[2] + size, ql[i] * g)] += 1
    return seen, rows, len(used)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl,hq,hk", [
    ([1], [1], 1, 1), ([1, 1, 1], [8192, 1, 700], 8, 2), ([0, 5, 0], [3, 0, 0], 4, 4), ([200, 33], [200, 900], 4, 1),
    ([300], [20], 5, 1), ([1000], [1000], 2, 2), ([100, 1], [5000, 129], 40, 8),
    ([64, 63, 257, 0], [64, 2000, 4100, 7], 2, 2), ([256], [3000], 1, 1)])
def test_plan_covers_every_pair_once(ql, kl, hq, hk, causal):
    plan = packed_plan(ql, kl, heads=hq, kv_heads=hk, head_dim=64, causal=causal, device="cpu")
    assert plan.total_q == sum(ql) and plan.total_k == sum(kl)
    g = hq // hk
    groups, shapes = (g, g, 1), ((16, 64), (64, 64), (256, 128))
    lists = [_covered(plan.tiles[i], plan.joins[i], groups[i], *shapes[i], ql, kl) for i in range(3)]
    assert [x[2] for x in lists] == list(plan.work.slots)
    assert plan.workspace_bytes == N.lib().vcattn_attn_packed_workspace_bytes(plan.work, hq, hk, 64)
    for i, (a, b) in enumerate(zip(ql, kl)):
        took = [(s[i], r[i], grp) for (s, r, _), grp in zip(lists, groups) if r[i].any()]
        assert len(took) == (1 if a else 0)
        for s, r, grp in took:
            assert (r == 1).all() and s.max(initial=0) <= 1
            for row in range(a * grp):
                lim = b if not causal else min(b, max(0, row // grp + 1 + b - a))
                assert (s[row, :lim] == 1).all()


def test_plan_refusals():
    for bad in (dict(q_lens=[-1]), dict(q_lens=[1], k_lens=[1, 2]), dict(q_lens=[1], heads=3, kv_heads=2),
                dict(q_lens=[1], head_dim=96), dict(q_lens=[2 ** 30, 2 ** 30, 5]), dict(q_lens=[1], heads=0)):
        args = dict(heads=2, head_dim=64, device="cpu")
        args.update(bad)
        with pytest.raises(ValueError):
            packed_plan(**args)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 4, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        qk_norm_rope(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_blocks(x)
    plan = packed_plan([4], heads=2, head_dim=64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(x.bfloat16(), x.bfloat16(), x.bfloat16(), plan)


def test_c_entry_points_check_their_arguments():
    lib = N.lib()
    P = 0x1000   # a pointer that no call here dereferences

    def view(p=P, s=64):
        return ctypes.byref(N.BHND(p, s, s, s))

    def rope(q=None, dtype=0, D=64, rot=32, flags=2, cos=P, sn=16, w=None):
        return lib.vcattn_qk_norm_rope(q or view(), view(), dtype, 1, 2, 2, 4, D, w, None, cos, cos, 0, sn, rot, flags,
                                       1e-5, view(), view(), None)

    for kw, text in ((dict(dtype=9), b"dtype"), (dict(D=60), b"multiple of 8"), (dict(rot=24), b"rot"),
                     (dict(flags=8), b"flag"), (dict(q=view(P + 2)), b"aligned"), (dict(cos=None), b"tables"),
                     (dict(sn=3), b"tables"), (dict(w=P + 4), b"weights"), (dict(q=view(None)), b"aligned")):
        assert rope(**kw) == N.ERR_ARG and text in lib.vcattn_last_error(), kw

    def quant(x=P, dtype=0, m=4, k=128, ldx=128, rows=1, codes=P, ldc=128, scale=P):
        return lib.vcattn_quantize_blocks(x, dtype, m, k, ldx, rows, codes, ldc, scale, 1, 4, None)

    for kw, text in ((dict(dtype=5), b"dtype"), (dict(rows=2), b"block_rows"), (dict(x=None), b"null"),
                     (dict(ldx=100), b"stride"), (dict(ldc=130), b"aligned"), (dict(m=-1), b"range")):
        assert quant(**kw) == N.ERR_ARG and text in lib.vcattn_last_error(), kw
    assert quant(m=0, x=None) == N.OK

    def mm(a=P, lda=128, m=4, n=8, k=128, dt=0, ldo=8, out=P, ldb=128):
        return lib.vcattn_matmul_blocks(a, lda, P, 1, 4, P, ldb, P, 1, 1, m, n, k, None, out, dt, ldo, None, 0, None)

    for kw, text in ((dict(a=None), b"null"), (dict(a=P + 1), b"aligned"), (dict(lda=100), b"aligned"), (dict(k=0), b"range"),
                     (dict(dt=7), b"dtype"), (dict(ldo=4), b"stride"), (dict(out=P + 1), b"misaligned")):
        assert mm(**kw) == N.ERR_ARG and text in lib.vcattn_last_error(), kw
    assert mm(m=0) == N.OK
    assert lib.vcattn_matmul_blocks_workspace_bytes(1000, 5376, 14336) == 20 * 7 * 128 * 256 * 4   # on 148 SMs
    assert mm(m=1000, n=5376, k=14336, lda=14336, ldb=14336, ldo=5376) == N.ERR_WORKSPACE
    assert lib.vcattn_matmul_blocks_workspace_bytes(1, 14336, 5376) == 0

    def attn(q=None, dtype=0, hq=4, hk=2, D=64, tiles=P, slots=0, scale=0.1, ws=None, wsb=0, n=1):
        work = N.PackedWork((None, tiles, None), (None,) * 3, (0, n, 0), (0, 0, 0), (0, slots, 0))
        return lib.vcattn_attn_packed(q or view(), view(), view(), dtype, hq, hk, 8, 8, D, work, 0, scale, view(),
                                      ws, wsb, None)

    for kw, text in ((dict(dtype=2), b"dtype"), (dict(hq=3), b"multiple"), (dict(D=96), b"D must"),
                     (dict(tiles=None), b"null"), (dict(scale=-1.0), b"scale"), (dict(q=view(P + 8)), b"aligned"),
                     (dict(n=-1), b"negative")):
        assert attn(**kw) == N.ERR_ARG and text in lib.vcattn_last_error(), kw
    assert attn(slots=3, ws=P, wsb=16) == N.ERR_WORKSPACE
    for name, call in (("vcattn_qk_norm_rope", rope), ("vcattn_quantize_blocks", quant), ("vcattn_matmul_blocks", mm),
                       ("vcattn_attn_packed", attn)):
        N.inject_fault(name)
        try:
            assert call() == N.ERR_INJECTED
        finally:
            N.inject_fault(None)
