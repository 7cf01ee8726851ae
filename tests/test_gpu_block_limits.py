"""Sizes past what the block operators' kernels index are refused before
anything is allocated or launched."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,hq,hk,n", [(1, 1, 0, 2 ** 32 + 1), (1, 1, 1, 2 ** 30), (2 ** 32, 1, 1, 1),
                                       (1, 2 ** 31, 2 ** 31, 1), (2 ** 16, 1, 0, 2 ** 16)])
def test_rope_of_2_to_the_31_rows(b, hq, hk, n):
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    x = torch.zeros(1, 1, 1, 8, device="cuda", dtype=torch.bfloat16)
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="2\\^31"):
        qk_norm_rope(x.expand(b, hq, n, 8), x[:, :0].expand(b, 0, n, 8) if hk == 0 else x.expand(b, hk, n, 8))
    assert torch.cuda.memory_allocated() == before
