"""The rotation tables of scaled positions, pair by pair (no GPU)."""

import math

import torch

from comfyui_vc_attention_b200.vc_attention import rope_tables


def test_yarn_between_the_bounds_is_linear_in_turns():
    """Every channel pair, the ones between beta_slow and beta_fast turns among them."""
    length, factor, fast, slow, dim = 4096, 8.0, 32.0, 1.0, 96
    cos, sin = rope_tables(torch.tensor([1, 977]), dim, 10000.0, scaling="yarn", factor=factor, original_len=length,
                           beta_fast=fast, beta_slow=slow)
    mult, between = 1 + 0.1 * math.log(factor), 0
    for i in range(dim // 2):
        inv = 10000.0 ** (-2 * i / dim)
        turns = length * inv / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
        between += 0 < keep < 1
        w = inv * keep + inv / factor * (1 - keep)
        for row, pos in enumerate((1, 977)):
            assert abs(cos[row, i].item() - mult * math.cos(pos * w)) < 2e-7
            assert abs(sin[row, i].item() - mult * math.sin(pos * w)) < 2e-7
    assert between > 10
