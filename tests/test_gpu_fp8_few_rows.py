"""matmul_blocks of 2 to 32 rows where several CTAs of a cluster share the
k-blocks of a tile, and where one CTA goes through more of them than its ring
holds.  Bounds as in test_gpu_fp8_linear."""

import pytest
import torch

from test_gpu_fp8_linear import _blocks, _check

pytestmark = pytest.mark.gpu

SIZES = [(16, 7168, 5376), (32, 7168, 5376), (17, 1000, 5376), (31, 130, 7184), (9, 640, 1040), (2, 5376, 7168),
         (16, 128, 14336), (32, 128, 14336), (25, 14336, 1296), (13, 43648, 1040), (29, 30336, 1040), (24, 20000, 2048)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, bias, dtype):
    from comfyui_vc_attention_b200.vc_attention import matmul_blocks
    a, b = _blocks(m, k, 1, m + n), _blocks(n, k, 128, k)
    x = torch.randn(n, device="cuda") if bias else None
    buf = torch.full((m + 2, n), 7.0, device="cuda", dtype=dtype)
    assert matmul_blocks(a, b, x, dtype, out=buf[1:-1]).data_ptr() == buf[1].data_ptr()
    _check(buf[1:-1], a, b, x)
    assert (buf[0] == 7).all() and (buf[-1] == 7).all()


@pytest.mark.parametrize("m", [2, 9, 16, 17, 32])
def test_the_same_bits_each_time(m):
    from comfyui_vc_attention_b200.vc_attention import matmul_blocks
    for n, k in ((7168, 5376), (130, 7184), (43648, 1040)):
        a, b = _blocks(m, k, 1, 1), _blocks(n, k, 128, 2)
        first = matmul_blocks(a, b)
        for _ in range(5):
            assert torch.equal(matmul_blocks(a, b), first)


def test_each_row_by_itself():
    """Rows of a product have the bits of the product of the row alone (same kernel, same ranks)."""
    from comfyui_vc_attention_b200.vc_attention import Fp8Blocks, matmul_blocks
    a, b = _blocks(16, 5376, 1, 5), _blocks(7168, 5376, 128, 6)
    whole = matmul_blocks(a, b, dtype=torch.float32)
    for i in (0, 7, 15):
        assert torch.equal(matmul_blocks(Fp8Blocks(a.codes[i:i + 1], a.scale[i:i + 1], 1), b, dtype=torch.float32)[0], whole[i])
