"""The block operators in a captured CUDA graph: replayed on new inputs they
give the bits of the direct calls (no call synchronises, and all buffers come
from torch's allocator)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_captured_block():
    from comfyui_vc_attention_b200.vc_attention import (linear_blocks, packed_attention, packed_plan, qk_norm_rope,
                                                        quantize_blocks, rope_tables)
    ql, kl, hq, hk, d = [130, 1, 20, 70], [130, 3000, 500, 70], 8, 2, 128
    g = torch.Generator("cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    w = quantize_blocks(r(hq * d, 512), rows=128)
    cos, sin = rope_tables(torch.arange(sum(ql)).cuda(), 96)
    x, k, v = r(sum(ql), 512), r(1, hk, sum(kl), d), r(1, hk, sum(kl), d)
    plan = packed_plan(ql, kl, heads=hq, kv_heads=hk, head_dim=d, causal=True)

    def step():
        q = linear_blocks(x, w).view(1, -1, hq, d).transpose(1, 2)
        q, _ = qk_norm_rope(q, q, cos, sin)
        return packed_attention(q, k, v, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.copy_(r(*x.shape))
        k.copy_(r(*k.shape))
        v.copy_(r(*v.shape))
        graph.replay()
        assert torch.equal(out, step())
