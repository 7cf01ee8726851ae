"""Argument checks of the block operators at the limits of their integer types (no GPU)."""

import ctypes

import numpy as np
import pytest
import torch

from comfyui_vc_attention_b200.vc_attention import _native as N, packed_plan

P = 0x1000   # a pointer that no call here dereferences


def test_rope_head_count_does_not_wrap():
    v = ctypes.byref(N.BHND(P, 64, 64, 64))
    for hq, hk, n in ((2 ** 30, 2 ** 30, 1), (2 ** 31 - 1, 1, 1), (1, 1, 2 ** 30)):
        rc = N.lib().vcattn_qk_norm_rope(v, v, 0, 1, hq, hk, n, 64, None, None, None, None, 0, 0, 0, 2, 1e-5, v, v, None)
        assert rc == N.ERR_ARG and b"2^31" in N.lib().vcattn_last_error(), (hq, hk, n)


def test_quantize_size_does_not_wrap():
    """2^60 rows of 16 blocks: the count of blocks is 0 modulo 2^64."""
    for m in (2 ** 60, 2 ** 62, 2 ** 63 - 1, 2 ** 36):
        for rows in (1, 128):
            rc = N.lib().vcattn_quantize_blocks(P, 0, m, 2048, 2048, rows, P, 2048, P, 1, 4, None)
            assert rc == N.ERR_ARG and b"range" in N.lib().vcattn_last_error(), (m, rows)


@pytest.mark.parametrize("bad", [[2 ** 62] * 4, [2 ** 63 - 1, 2 ** 63 - 1, 2], [2 ** 64], [2 ** 31], [2 ** 30] * 2])
def test_plan_lengths_that_add_up_past_64_bits(bad):
    for kw in (dict(q_lens=bad), dict(q_lens=[1] * len(bad), k_lens=bad)):
        with pytest.raises(ValueError, match="2\\^31"):
            packed_plan(heads=1, head_dim=64, device="cpu", **kw)


@pytest.mark.parametrize("bad", [[2.7], ["3"], [None], [1, 2.0]])
def test_plan_lengths_that_are_no_whole_numbers(bad):
    for kw in (dict(q_lens=bad), dict(q_lens=[1] * len(bad), k_lens=bad)):
        with pytest.raises(TypeError, match="whole"):
            packed_plan(heads=1, head_dim=64, device="cpu", **kw)


def test_plan_lengths_of_other_integer_types():
    for lens in ((3, 5), np.array([3, 5], dtype=np.int32), torch.tensor([3, 5]), [np.uint8(3), torch.tensor(5)]):
        assert packed_plan(lens, heads=1, head_dim=64, device="cpu").total_q == 8
