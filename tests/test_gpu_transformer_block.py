"""The operators together, as examples/transformer_block.py runs them, against
the same block in 64 bits on the unquantised weights.

E4M3 keeps four significant bits, so each projection's inputs and weights are
off by at most 2^-4 of a value and, being rounded to nearest, by about 2.6 % in
the mean square each; the block's output then differs by a few per cent in the
2-norm.  Wrong heads, positions, masks or scales differ by the norm itself."""

import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def _exact(block, x, cos, sin, lens, causal):
    h, hk, d = block.heads, block.kv_heads, block.head_dim
    qkv = (x.double() @ block.w_qkv.double().t()).view(x.shape[0], -1, d)
    c, s, r = cos.double()[:, None], sin.double()[:, None], cos.shape[-1]

    def turn(y, w):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        a, b = y[..., :r].clone(), y[..., r:2 * r].clone()
        y[..., :r], y[..., r:2 * r] = a * c - b * s, b * c + a * s
        return y

    q, k, v = turn(qkv[:, :h], block.q_norm), turn(qkv[:, h:h + hk], block.k_norm), qkv[:, h + hk:]
    k, v = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
    out, at = torch.empty_like(q), 0
    for n in lens:
        i = slice(at, at + n)
        sc = torch.einsum("qhd,khd->hqk", q[i], k[i]) / math.sqrt(d)
        if causal:
            sc = sc.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        out[i] = torch.einsum("hqk,khd->qhd", sc.softmax(-1), v[i])
        at += n
    return out.reshape(x.shape[0], -1) @ block.w_out.double().t()


def test_prompts():
    from transformer_block import AttentionBlock
    from comfyui_vc_attention_b200.vc_attention import packed_plan, rope_tables
    block, lens = AttentionBlock(heads=8, kv_heads=2), [77, 300, 1, 128]
    cos, sin = rope_tables(torch.cat([torch.arange(n) for n in lens]).cuda(), 96)
    x = torch.randn(sum(lens), 1024, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    plan = packed_plan(lens, heads=8, kv_heads=2, head_dim=128, causal=True)
    y, ref = block.prompts(x, cos, sin, plan), _exact(block, x, cos, sin, lens, True)
    assert ((y.double() - ref).norm() / ref.norm()).item() < 0.15


def test_clip():
    from transformer_block import AttentionBlock
    from comfyui_vc_attention_b200.vc_attention import rope_tables
    block, n = AttentionBlock(heads=4), 2048
    cos, sin = rope_tables(torch.arange(n).cuda(), 96)
    x = torch.randn(n, 1024, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(torch.bfloat16)
    y, ref = block.clip(x, cos, sin), _exact(block, x, cos, sin, [n], False)
    assert y.shape == ref.shape and torch.isfinite(y).all()
    assert ((y.double() - ref).norm() / ref.norm()).item() < 0.25


def test_main_runs(capsys):
    import transformer_block
    transformer_block.main()
    assert "prompts:" in capsys.readouterr().out
