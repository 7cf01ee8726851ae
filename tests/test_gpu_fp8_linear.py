"""quantize_blocks bit for bit against IEEE fp32 arithmetic, and matmul_blocks
against 64-bit sums.

Tolerance of the product: E4M3 products are exact; a 128-column block sum takes
four MMAs of 32 columns with fp32 accumulation (at most 33 roundings of 2^-23
each, relative to the sum of the magnitudes), each block one scaled addition.
Then one rounding to the output type (2^-8 bf16, 2^-11 fp16).
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _e4m3_values():
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))


def _nearest_code(q):
    """Codes 0..126 of |q| (round to nearest, ties to the even code), the sign of q < 0 in bit 7."""
    v = _e4m3_values()
    a = np.minimum(np.abs(q.astype(np.float64)), 448.0)
    hi = np.clip(np.searchsorted(v, a), 1, 126)
    lo = hi - 1
    dl, dh = a - v[lo], v[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return np.where(q < 0, code + 128, code).astype(np.uint8)


def _quant_oracle(x, rows):
    m, k = x.shape
    kb, mb = -(-k // 128), -(-m // rows)
    pad = np.zeros((mb * rows, kb * 128), dtype=np.float32)
    pad[:m, :k] = x
    f = pad.reshape(mb, rows, kb, 128)
    s = np.maximum(np.abs(f).max((1, 3)), np.float32(1e-30)) / np.float32(448)
    q = (f / s[:, None, :, None]).reshape(mb * rows, kb * 128)[:m, :k]
    return _nearest_code(q), s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (130, 129), (257, 5376), (2, 14336), (128, 256), (5, 300)])
def test_codes_and_scales_are_exact(dtype, rows, m, k):
    from comfyui_vc_attention_b200.vc_attention import quantize_blocks
    torch.manual_seed(m * k)
    x = (torch.randn(m, k, device="cuda") * torch.exp(2 * torch.randn(m, 1, device="cuda"))).to(dtype)
    x[:, k // 2] = 0
    b = quantize_blocks(x, rows)
    codes, scale = _quant_oracle(x.float().cpu().numpy(), rows)
    assert b.codes.shape == (m, k) and b.codes.dtype == torch.float8_e4m3fn and b.rows == rows
    assert np.array_equal(b.scale.cpu().numpy(), scale)
    assert np.array_equal(b.codes.contiguous().view(torch.uint8).cpu().numpy(), codes)


def test_quantise_strides_leading_dims_and_special_values():
    from comfyui_vc_attention_b200.vc_attention import quantize_blocks
    base = torch.randn(6, 515, device="cuda").to(torch.bfloat16)
    for x in (base[:, 3:259], base[::2, :256], base.t()[:256].t(), base[:1, 1:]):
        b = quantize_blocks(x)
        codes, scale = _quant_oracle(x.float().cpu().numpy(), 1)
        assert np.array_equal(b.codes.contiguous().view(torch.uint8).cpu().numpy(), codes)
        assert np.array_equal(b.scale.cpu().numpy(), scale)
    x3 = torch.randn(2, 3, 256, device="cuda")
    assert torch.equal(quantize_blocks(x3).scale, quantize_blocks(x3.view(6, 256)).scale)
    x = torch.ones(4, 256, device="cuda")
    x[0, 0], x[1, 0], x[2, :128], x[3, :] = float("inf"), float("nan"), 0.0, 1e-38
    b = quantize_blocks(x)
    v = b.codes.float()
    assert b.scale[0, 0].isinf() and v[0, 0].isnan() and (v[0, 1:128] == 0).all() and (v[0, 128:] == 448).all()
    assert b.scale[1, 0].isnan() and v[1, :128].isnan().all() and (v[1, 128:] == 448).all()
    assert (v[2, :128] == 0).all() and torch.isfinite(b.scale[2]).all()
    assert torch.isfinite(v[3]).all()
    assert quantize_blocks(torch.empty(0, 256, device="cuda")).codes.shape == (0, 256)


def _blocks(m, k, rows, seed):
    from comfyui_vc_attention_b200.vc_attention import Fp8Blocks
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = (100 * torch.randn(m, k, generator=g, device="cuda")).clamp_(-448, 448).to(torch.float8_e4m3fn)
    s = torch.exp(torch.randn(-(-k // 128), -(-m // rows), generator=g, device="cuda")).mul_(0.01).t()
    return Fp8Blocks(c, s, rows)


def _dequant(b):
    m, k = b.codes.shape
    s = b.scale.double().repeat_interleave(b.rows, 0)[:m].repeat_interleave(128, 1)[:, :k]
    return b.codes.double() * s


def _check(out, a, b, bias):
    x, y = _dequant(a), _dequant(b)
    ref, size = x @ y.t(), x.abs() @ y.abs().t()
    if bias is not None:
        ref, size = ref + bias.double(), size + bias.double().abs()
    kb = -(-a.codes.shape[1] // 128)
    bound = HALF_UNIT[out.dtype] * ref.abs() + (4 * 33 + kb + 4) * 2.0 ** -23 * size
    bad = (out.double() - ref).abs() > 1.01 * bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound"
    # and the typical error is that of the rounding, not of the bound
    rel = ((out.double() - ref).norm() / ref.norm()).item()
    assert rel < max(HALF_UNIT[out.dtype], 2e-6), rel


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [
    (1, 128, 128), (1, 5376, 7168), (2, 8, 16), (7, 200, 304), (16, 1, 128), (17, 129, 256), (33, 384, 1040),
    (64, 1000, 512), (65, 640, 2048), (129, 257, 144), (128, 256, 128), (333, 1536, 640), (1000, 5376, 384),
    (2100, 2304, 256), (1, 3, 5376), (1000, 5376, 6272), (1021, 5302, 6400)])
def test_product(dtype, m, n, k):
    from comfyui_vc_attention_b200.vc_attention import matmul_blocks
    a, b = _blocks(m, k, 1, 1), _blocks(n, k, 128, 2)
    bias = torch.randn(n, device="cuda") if n % 2 == 0 else None
    _check(matmul_blocks(a, b, bias, dtype), a, b, bias)


def test_product_views_and_ragged_k():
    from comfyui_vc_attention_b200.vc_attention import Fp8Blocks, matmul_blocks, quantize_blocks
    # K that is no multiple of 16: quantize_blocks pads the pitch, foreign codes are copied
    a, b = quantize_blocks(torch.randn(37, 203, device="cuda")), quantize_blocks(torch.randn(150, 203, device="cuda"), 128)
    _check(matmul_blocks(a, b, dtype=torch.float32), a, b, None)
    a2, b2 = (Fp8Blocks(x.codes.contiguous(), x.scale.contiguous(), x.rows) for x in (a, b))   # other scale order
    assert torch.equal(matmul_blocks(a2, b2, dtype=torch.float32), matmul_blocks(a, b, dtype=torch.float32))
    # output into a column slice with an odd offset: nothing beside it changes
    buf = torch.full((37, 401), 7.0, device="cuda", dtype=torch.bfloat16)
    matmul_blocks(a, b, out=buf[:, 3:153])
    _check(buf[:, 3:153], a, b, None)
    assert (buf[:, :3] == 7).all() and (buf[:, 153:] == 7).all()
    # rows past M and N are not read as values: codes of a larger buffer hold NaN there
    big = torch.full((64, 256), float("nan"), device="cuda").to(torch.float8_e4m3fn)
    big[:5] = _blocks(5, 256, 1, 3).codes
    a, b = Fp8Blocks(big[:5], _blocks(5, 256, 1, 3).scale, 1), _blocks(40, 256, 128, 4)
    _check(matmul_blocks(a, b), a, b, None)
    assert matmul_blocks(_blocks(0, 256, 1, 0), b).shape == (0, 40)


def test_repeated_calls_give_the_same_bits_and_streams():
    from comfyui_vc_attention_b200.vc_attention import matmul_blocks
    for m in (1, 40, 700):
        a, b = _blocks(m, 5376, 1, 1), _blocks(1536, 5376, 128, 2)
        first = matmul_blocks(a, b)
        for _ in range(3):
            assert torch.equal(matmul_blocks(a, b), first)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = matmul_blocks(a, b)
        s.synchronize()
        assert torch.equal(other, first)


def test_linear_blocks():
    from comfyui_vc_attention_b200.vc_attention import linear_blocks, matmul_blocks, quantize_blocks
    x = torch.randn(2, 19, 640, device="cuda").to(torch.bfloat16)
    w = torch.randn(384, 640, device="cuda").to(torch.bfloat16) / 25
    wq, bias = quantize_blocks(w, rows=128), torch.randn(384, device="cuda")
    y = linear_blocks(x, wq, bias)
    assert y.shape == (2, 19, 384) and y.dtype == torch.bfloat16
    assert torch.equal(y.view(38, 384), matmul_blocks(quantize_blocks(x.view(38, 640)), wq, bias))
    ref = x.double().view(38, 640) @ w.double().t() + bias.double()
    # E4M3 keeps 4 significant bits: each factor is off by at most 2^-4 relative
    size = x.double().view(38, 640).abs() @ w.double().abs().t()
    assert ((y.view(38, 384).double() - ref).abs() <= 0.13 * size + 2.0 ** -8 * ref.abs()).all()


def test_refusals():
    from comfyui_vc_attention_b200.vc_attention import Fp8Blocks, matmul_blocks, quantize_blocks
    a, b = _blocks(4, 256, 1, 1), _blocks(130, 256, 128, 2)
    for bad in (lambda: quantize_blocks(torch.randn(4, 4, device="cuda"), rows=64),
                lambda: quantize_blocks(torch.ones(4, 4, device="cuda", dtype=torch.int32)),
                lambda: quantize_blocks(torch.empty(4, 0, device="cuda")),
                lambda: matmul_blocks(b, b), lambda: matmul_blocks(a, a),
                lambda: matmul_blocks(a, _blocks(130, 128, 128, 2)),
                lambda: matmul_blocks(Fp8Blocks(a.codes, a.scale[:, :1], 1), b),
                lambda: matmul_blocks(Fp8Blocks(a.codes, a.scale.double(), 1), b),
                lambda: matmul_blocks(Fp8Blocks(a.codes.view(torch.uint8), a.scale, 1), b),
                lambda: matmul_blocks(a, b, torch.ones(129, device="cuda")),
                lambda: matmul_blocks(a, b, torch.ones(130)),
                lambda: matmul_blocks(a, b, dtype=torch.int32),
                lambda: matmul_blocks(a, b, out=torch.empty(4, 129, device="cuda", dtype=torch.bfloat16)),
                lambda: matmul_blocks(a, b, out=torch.empty(130, 4, device="cuda", dtype=torch.bfloat16).t())):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(RuntimeError):
        quantize_blocks(torch.ones(4, 128))
    with pytest.raises(RuntimeError, match="no backward"):
        quantize_blocks(torch.ones(4, 128, device="cuda", requires_grad=True))
