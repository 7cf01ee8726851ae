"""The block operators have no derivatives and say so, before anything else is
looked at (no GPU)."""

import pytest
import torch
from torch.autograd import forward_ad

from comfyui_vc_attention_b200.vc_attention import (Fp8Blocks, matmul_blocks, packed_attention, packed_plan,
                                                    qk_norm_rope, quantize_blocks)


def _calls():
    """Name, tensors, and the call on them."""
    x, t, w = torch.randn(1, 2, 4, 64), torch.randn(4, 16), torch.randn(64)
    yield "qk_norm_rope", [x, x.clone(), t, t.clone(), w, w.clone(), x.clone(), x.clone()], \
        lambda q, k, c, s, a, b, oq, ok: qk_norm_rope(q, k, c, s, a, b, out=(oq, ok))
    yield "quantize_blocks", [torch.randn(4, 128)], quantize_blocks
    a8, b8 = torch.randn(4, 128).to(torch.float8_e4m3fn), torch.randn(8, 128).to(torch.float8_e4m3fn)
    yield "matmul_blocks", [a8, torch.ones(4, 1), b8, torch.ones(1, 1), torch.ones(8), torch.empty(4, 8)], \
        lambda a, sa, b, sb, bias, out: matmul_blocks(Fp8Blocks(a, sa, 1), Fp8Blocks(b, sb, 128), bias, torch.float32, out)
    plan = packed_plan([4], heads=2, head_dim=64, device="cpu")
    y = x.bfloat16()
    yield "packed_attention", [y, y.clone(), y.clone(), y.clone()], lambda q, k, v, o: packed_attention(q, k, v, plan, out=o)


CASES = [(name, i) for name, tensors, _ in _calls() for i in range(len(tensors))]


def _case(name):
    return next((t, f) for n, t, f in _calls() if n == name)


@pytest.mark.parametrize("name,i", CASES)
def test_a_tensor_that_requires_a_gradient(name, i):
    tensors, call = _case(name)
    tensors[i].requires_grad_()
    with pytest.raises(RuntimeError, match=name + " has no backward"):
        call(*tensors)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        call(*tensors)


@pytest.mark.parametrize("name,i", [c for c in CASES if c not in (("matmul_blocks", 0), ("matmul_blocks", 2))])
def test_a_dual_tensor(name, i):
    tensors, call = _case(name)
    with forward_ad.dual_level():
        tensors[i] = forward_ad.make_dual(tensors[i], torch.ones_like(tensors[i]))
        with pytest.raises(RuntimeError, match=name + " has no forward"):
            call(*tensors)
        with torch.no_grad(), pytest.raises(RuntimeError, match=name + " has no forward"):
            call(*tensors)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(*tensors)
