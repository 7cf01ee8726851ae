"""quantize_blocks bit for bit against IEEE fp32 divisions where the block's
maximum is tiny: values next to the ties of the codes, whose quotients'
remainders are below the fp32 subnormal step."""

import numpy as np
import pytest
import torch

from test_gpu_fp8_linear import _e4m3_values, _quant_oracle

pytestmark = pytest.mark.gpu


def _near_ties(rows, k, exponents, seed):
    """Rows of `k` columns: the first holds the maximum, the others lie within two fp32
    steps of a tie between two codes."""
    g = np.random.default_rng(seed)
    top = np.maximum((g.uniform(1, 2, rows) * 2.0 ** g.choice(exponents, rows)).astype(np.float32), np.float32(1e-30))
    v = _e4m3_values()
    tie = g.choice((v[1:] + v[:-1]) / 2, (rows, k)) * g.choice([-1.0, 1.0], (rows, k))
    x = (tie * (top / np.float32(448)).astype(np.float64)[:, None]).astype(np.float32)
    x = (x.view(np.int32) + g.integers(-2, 3, x.shape).astype(np.int32)).view(np.float32)
    x[:, ::128] = top[:, None]
    return x


@pytest.mark.parametrize("low,high", [(-100, -98), (-99, -94), (-95, -88), (-92, -80), (-60, 60)])
def test_codes_of_tiny_blocks(low, high):
    from comfyui_vc_attention_b200.vc_attention import quantize_blocks
    x = _near_ties(4096, 512, np.arange(low, high), seed=200 + high)
    b = quantize_blocks(torch.from_numpy(x).cuda())
    codes, scale = _quant_oracle(x, 1)
    assert np.array_equal(b.scale.cpu().numpy(), scale)
    got = b.codes.view(torch.uint8).cpu().numpy()
    assert np.array_equal(got, codes), f"{int((got != codes).sum())} of {codes.size} codes"


def test_pinned_value():
    """max 0x1.bfe5d4p-99, x 0x1.ffe218p-118: a code that the rounded remainder gets wrong."""
    from comfyui_vc_attention_b200.vc_attention import quantize_blocks
    x = np.zeros((130, 128), dtype=np.float32)
    x[:, 0], x[:, 1], x[:, 2] = (float.fromhex(h) for h in ("0x1.bfe5d4p-99", "0x1.ffe218p-118", "-0x1.ffe218p-118"))
    for rows in (1, 128):
        codes, scale = _quant_oracle(x, rows)
        b = quantize_blocks(torch.from_numpy(x).cuda(), rows)
        assert np.array_equal(b.scale.cpu().numpy(), scale)
        assert np.array_equal(b.codes.view(torch.uint8).cpu().numpy(), codes)
    z = torch.zeros(130, 300, device="cuda")
    assert (quantize_blocks(z).codes.float() == 0).all() and (quantize_blocks(z, 128).codes.float() == 0).all()
