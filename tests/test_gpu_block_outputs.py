"""Outputs that the caller gives: over the input where that is defined, refused
where they would be read and written by different threads."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _tables(n, rot):
    a = torch.rand(n, rot // 2, device="cuda") * 6
    return a.cos(), a.sin()


def test_rope_outputs_that_overlap():
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    q, k = (torch.randn(1, 4, 300, 64, device="cuda").to(torch.bfloat16) for _ in range(2))
    cos, sin = _tables(300, 64)
    both = torch.empty(2, 1, 4, 300, 64, device="cuda", dtype=torch.bfloat16)
    flat = both.view(-1)
    n = q.numel()
    for out in ((k, q), (k, both[0]), (both[0], q), (both[0], both[0]), (q, q),
                (flat[:n].view_as(q), flat[n // 2:n // 2 + n].view_as(q))):
        with pytest.raises(ValueError, match="overlaps"):
            qk_norm_rope(q, k, cos, sin, out=out)
    with pytest.raises(ValueError, match="overlaps"):                       # one tensor as both, in place
        qk_norm_rope(q, q, cos, sin, out=(q, torch.empty_like(q)))
    part = torch.empty(n + 512, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="part"):
        qk_norm_rope(part[:n].view_as(q), k, cos, sin, out=(part[512:].view_as(q), both[0]))
    # views of one projection: swapped, and in place
    qkv = torch.randn(1, 300, 12, 64, device="cuda").to(torch.bfloat16)
    q, k = qkv[:, :, :4].transpose(1, 2), qkv[:, :, 4:8].transpose(1, 2)
    with pytest.raises(ValueError, match="overlaps"):
        qk_norm_rope(q, k, cos, sin, out=(k, q))
    want = qk_norm_rope(q, k, cos, sin)
    qk_norm_rope(q, k, cos, sin, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_attention_outputs_that_overlap():
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v = (torch.randn(1, 4, 300, 64, device="cuda").to(torch.bfloat16) for _ in range(3))
    plan = packed_plan([300], heads=4, head_dim=64, causal=True)
    want = packed_attention(q, k, v, plan)
    for out in (k, v):
        with pytest.raises(ValueError, match="overlaps"):
            packed_attention(q, k, v, plan, out=out)
    assert torch.equal(packed_attention(q, k, v, plan), want)
    assert torch.equal(packed_attention(q, k, v, plan, out=q), want)        # over q


def test_product_outputs_that_overlap():
    from comfyui_vc_attention_b200.vc_attention import Fp8Blocks, matmul_blocks
    store = torch.zeros(300 * 512 * 4, dtype=torch.uint8, device="cuda")
    a = Fp8Blocks(store[:40 * 256].view(torch.float8_e4m3fn).view(40, 256), torch.ones(40, 2, device="cuda"), 1)
    b = Fp8Blocks(torch.zeros(128, 256, device="cuda").to(torch.float8_e4m3fn), torch.ones(1, 2, device="cuda"), 128)
    with pytest.raises(ValueError, match="overlaps"):
        matmul_blocks(a, b, out=store[:40 * 128 * 2].view(torch.bfloat16).view(40, 128))
    y = torch.empty(40, 128, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        matmul_blocks(a, b, y[0], torch.float32, out=y)
    matmul_blocks(a, b, out=store[40 * 256:40 * 256 + 40 * 128 * 2].view(torch.bfloat16).view(40, 128))


@pytest.mark.parametrize("d,lq,lk", [(128, 300, 300), (64, 300, 300), (128, 270, 5000), (128, 30, 90), (64, 4, 700)])
def test_attention_over_q_with_infinite_values(d, lq, lk):
    """Values that are infinite behind the causal mask of some rows, in channels of several
    parts of the row: the output over q has the bits of the output beside it."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    g = torch.Generator("cuda").manual_seed(d + lk)
    q, k, v = (torch.randn(1, 8, n, d, generator=g, device="cuda").to(torch.bfloat16) for n in (lq, lk, lk))
    for i, c in enumerate((3, 40, d - 1, 17, 33)):
        v[:, :, lk - lq + (i + 1) * lq // 7, c] = float("inf") if i % 2 else -float("inf")
        v[:, :, lk - lq + (i + 1) * lq // 7, (c + 32) % d] = float("inf")
    plan = packed_plan([lq], [lk], heads=8, head_dim=d, causal=True)
    want = packed_attention(q, k, v, plan)
    assert want.isinf().any() and torch.isfinite(want).any()
    got = packed_attention(q, k, v, plan, out=q)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_autograd_sees_what_was_written():
    """A backward pass that needs a tensor which an operator has overwritten refuses."""
    from comfyui_vc_attention_b200.vc_attention import (matmul_blocks, packed_attention, packed_plan, qk_norm_rope,
                                                        quantize_blocks)
    cos, sin = _tables(20, 64)
    plan = packed_plan([20], heads=2, head_dim=64)
    a8 = quantize_blocks(torch.randn(10, 128, device="cuda"))
    b8 = quantize_blocks(torch.randn(256, 128, device="cuda"), 128)
    calls = [lambda x: qk_norm_rope(x, x.clone(), cos, sin, out=(x, x.clone())),
             lambda x: qk_norm_rope(x.clone(), x, cos, sin, out=(x.clone(), x)),
             lambda x: packed_attention(x, x.clone(), x.clone(), plan, out=x),
             lambda x: matmul_blocks(a8, b8, dtype=x.dtype, out=x.view(10, 256))]
    for call in calls:
        w = torch.ones(1, 2, 20, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = w * 1
        z = (y * y).sum()
        call(y.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    with torch.inference_mode():
        x = torch.ones(1, 2, 20, 64, device="cuda", dtype=torch.bfloat16)
        for call in calls:
            call(x)
