"""Argument checks of the block operators at the limits of their integer types (no GPU)."""

import ctypes

from comfyui_vc_attention_b200.vc_attention import _native as N

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
