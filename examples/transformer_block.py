"""One attention block of a DiT on this package's operators.

    hidden -> QKV projection (linear_blocks, 8-bit)
           -> RMS norm of q and k heads + rotation (qk_norm_rope, strided views of the projection)
           -> attention: packed_attention for prompts and short sequences,
              vc_attention_cuda for one long clip
           -> output projection (linear_blocks)

Run on a B200:  python examples/transformer_block.py
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from comfyui_vc_attention_b200.vc_attention import (build_permutation, packed_attention, packed_plan,  # noqa: E402
                                                    qk_norm_rope, quantize_blocks, linear_blocks, rope_tables,
                                                    GroupingConfig, H3, vc_attention_cuda)


class AttentionBlock:
    """Weights of one block, quantised once."""

    def __init__(self, hidden=1024, heads=8, kv_heads=None, head_dim=128, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads or heads, head_dim
        rows = (heads + 2 * self.kv_heads) * head_dim
        self.w_qkv = torch.randn(rows, hidden, generator=g, device=device).to(torch.bfloat16) / hidden ** 0.5
        self.w_out = torch.randn(hidden, heads * head_dim, generator=g, device=device).to(torch.bfloat16) / hidden ** 0.5
        self.q_norm = 1 + 0.1 * torch.randn(head_dim, generator=g, device=device)
        self.k_norm = 1 + 0.1 * torch.randn(head_dim, generator=g, device=device)
        self.qkv8, self.out8 = quantize_blocks(self.w_qkv, rows=128), quantize_blocks(self.w_out, rows=128)

    def project(self, x, cos, sin):
        """(1, H, T, D) q, k, v of the rows x (T, hidden); q and k normed and rotated."""
        t = x.shape[0]
        qkv = linear_blocks(x, self.qkv8).view(1, t, -1, self.head_dim)
        q, k, v = (s.transpose(1, 2) for s in qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=2))
        q, k = qk_norm_rope(q, k, cos, sin, self.q_norm, self.k_norm, eps=H3.qk_norm_eps)
        return q, k, v

    def finish(self, o):
        return linear_blocks(o.transpose(1, 2).reshape(o.shape[2], -1), self.out8)

    def prompts(self, x, cos, sin, plan):
        """Packed sequences of different lengths, exact attention."""
        q, k, v = self.project(x, cos, sin)
        return self.finish(packed_attention(q, k, v, plan))

    def clip(self, x, cos, sin):
        """One long sequence, VC-Attention."""
        q, k, v = self.project(x, cos, sin)
        perm = build_permutation(v[0], GroupingConfig(block_rows=128)).perm
        return self.finish(vc_attention_cuda(q, k, v, perm=perm))


def main():
    block = AttentionBlock(heads=8, kv_heads=2)
    lens = [77, 300, 1, 128]
    pos = torch.cat([torch.arange(n) for n in lens]).cuda()
    cos, sin = rope_tables(pos, H3.rope_dims)
    plan = packed_plan(lens, heads=8, kv_heads=2, head_dim=128, causal=True)
    y = block.prompts(torch.randn(sum(lens), 1024, device="cuda").to(torch.bfloat16), cos, sin, plan)
    print("prompts:", lens, "->", tuple(y.shape), y.dtype)

    block = AttentionBlock()
    t, h, w = 16, 16, 32                             # one clip's latent grid, rotated along three axes
    grid = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(h), torch.arange(w), indexing="ij"), -1)
    axis = 2 * H3.rope_freq_dim
    cos, sin = rope_tables(grid.view(-1, 3).cuda(), (axis, axis, axis))
    y = block.clip(torch.randn(t * h * w, 1024, device="cuda").to(torch.bfloat16), cos, sin)
    print("clip:", (t, h, w), "->", tuple(y.shape), y.dtype)


if __name__ == "__main__":
    main()
