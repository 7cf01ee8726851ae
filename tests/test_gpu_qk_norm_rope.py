"""qk_norm_rope against the formula in 64 bits.

Tolerance: the kernel works in fp32 (a row's sum of squares, one rsqrt, two
products and a sum per channel: at most 8 roundings of 2^-24 relative to the
larger of the pair) and rounds once to the output type (half a unit: 2^-8 for
bf16, 2^-11 for fp16, and 2^-25 absolute below its normal range).
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _exact(x, w, cos, sin, rot, layout, eps, norm):
    x = x.double()
    y = x if not norm else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    size = y.abs()
    if rot:
        c, s = cos.double(), sin.double()
        if c.dim() == 3:
            c, s = c[:, None], s[:, None]
        h = rot // 2
        i, j = (slice(0, h), slice(h, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
        y1, y2 = y[..., i].clone(), y[..., j].clone()
        y[..., i], y[..., j] = y1 * c - y2 * s, y2 * c + y1 * s
        size[..., i] = size[..., j] = y1.abs() + y2.abs()
    return y, size


def _check(got, x, w, cos, sin, rot, layout, eps, norm):
    ref, size = _exact(x, w, cos, sin, rot, layout, eps, norm)
    u = HALF_UNIT[x.dtype]
    bound = u * ref.abs() + 8 * 2.0 ** -24 * size + (2.0 ** -25 if x.dtype == torch.float16 else 1e-30)
    bad = (got.double() - ref).abs() > bound * 1.01
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} channels outside the bound"


def _tables(n, rot, b=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (n, rot // 2) if b is None else (b, n, rot // 2)
    a = torch.rand(shape, generator=g, device="cuda", dtype=torch.float64) * 6.3
    return a.cos().float(), a.sin().float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("b,n,hq,hk,d,rot", [
    (1, 1, 1, 1, 64, 64), (1, 1, 32, 8, 128, 128), (2, 333, 5, 1, 64, 32), (1, 7, 56, 56, 128, 96),
    (3, 17, 9, 3, 128, 16), (1, 5, 4, 2, 256, 256), (2, 3, 3, 3, 96, 48), (1, 2, 2, 1, 8, 0), (1, 4, 2, 2, 72, 64)])
def test_matches_formula(dtype, layout, b, n, hq, hk, d, rot):
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    torch.manual_seed(n + d)
    q = (3 * torch.randn(b, hq, n, d, device="cuda")).to(dtype)
    k = torch.randn(b, hk, n, d, device="cuda").to(dtype)
    qw, kw = torch.randn(d, device="cuda"), 1 + 0.1 * torch.randn(d, device="cuda")
    cos, sin = _tables(n, rot) if rot else (None, None)
    oq, ok = qk_norm_rope(q, k, cos, sin, qw, kw, layout=layout, eps=1e-5)
    _check(oq, q, qw, cos, sin, rot, layout, 1e-5, True)
    _check(ok, k, kw, cos, sin, rot, layout, 1e-5, True)


@pytest.mark.parametrize("norm", [True, False])
def test_without_weights_and_without_norm(norm):
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    q, k = torch.randn(1, 3, 9, 128, device="cuda"), torch.randn(1, 1, 9, 128, device="cuda")
    cos, sin = _tables(9, 96)
    oq, ok = qk_norm_rope(q, k, cos, sin, norm=norm)
    _check(oq, q, None, cos, sin, 96, "half", 1e-5, norm)
    _check(ok, k, None, cos, sin, 96, "half", 1e-5, norm)


def test_fused_projection_views_and_table_per_batch_entry():
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    b, n, hq, hk, d = 2, 45, 8, 2, 128
    qkv = torch.randn(b, n, hq + 2 * hk, d, device="cuda").to(torch.bfloat16)
    keep = qkv.clone()
    q, k = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hk].transpose(1, 2)
    cos, sin = _tables(n, 64, b)
    oq, ok = qk_norm_rope(q, k, cos, sin)
    _check(oq, q, None, cos, sin, 64, "half", 1e-5, True)
    _check(ok, k, None, cos, sin, 64, "half", 1e-5, True)
    assert torch.equal(qkv, keep)
    assert oq.transpose(1, 2).is_contiguous()
    # in place: the views are overwritten, v and nothing else is untouched
    qk_norm_rope(q, k, cos, sin, out=(q, k))
    assert torch.equal(q, oq) and torch.equal(k, ok)
    assert torch.equal(qkv[:, :, hq + hk:], keep[:, :, hq + hk:])


def test_unaligned_and_reordered_inputs():
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    cos, sin = _tables(6, 64)
    flat = torch.randn(2 * 6 * 3 * 64 + 1, device="cuda").to(torch.float16)
    q = flat[1:].view(2, 3, 6, 64)                                                   # 2-byte aligned
    k = torch.randn(64, 6, 3, 2, device="cuda").to(torch.float16).permute(3, 2, 1, 0)  # channels not contiguous
    w = torch.randn(65, device="cuda")[1:]
    big = torch.randn(6, 65, device="cuda")
    for c, s in ((cos, sin), (big[:, 1:33], big[:, 33:65])):
        oq, ok = qk_norm_rope(q, k, c, s, w, w)
        _check(oq, q, w, c, s, 64, "half", 1e-5, True)
        _check(ok, k, w, c, s, 64, "half", 1e-5, True)


def test_zero_rows_infinities_and_empty():
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    cos, sin = _tables(3, 64)
    q = torch.zeros(1, 2, 3, 128, device="cuda")
    k = torch.ones(1, 1, 3, 128, device="cuda")
    k[0, 0, 1, 0], k[0, 0, 2, 5] = float("inf"), float("nan")
    oq, ok = qk_norm_rope(q, k, cos, sin)
    assert torch.equal(oq, torch.zeros_like(oq))
    assert torch.isfinite(ok[0, 0, 0]).all() and ok[0, 0, 2].isnan().all()
    assert ok[0, 0, 1, [0, 32]].isnan().all() and (ok[0, 0, 1, 64:] == 0).all()
    # without the norm an infinite channel reaches only its own pair
    _, ok = qk_norm_rope(q, k, cos, sin, norm=False)
    assert torch.isfinite(ok[0, 0, 1, 64:]).all() and torch.isfinite(ok[0, 0, 1, 1:32]).all()
    e = torch.empty(1, 2, 0, 64, device="cuda")
    oq, ok = qk_norm_rope(e, e, *_tables(0, 32))
    assert oq.shape == e.shape and ok.shape == e.shape


def test_other_stream():
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    q = torch.randn(1, 8, 2048, 128, device="cuda").to(torch.bfloat16)
    cos, sin = _tables(2048, 128)
    want = qk_norm_rope(q, q, cos, sin)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = qk_norm_rope(q, q, cos, sin)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    from comfyui_vc_attention_b200.vc_attention import qk_norm_rope
    q = torch.randn(1, 2, 4, 64, device="cuda")
    cos, sin = _tables(4, 32)
    for bad in (dict(q=q[0]), dict(k=q[:, :, :3]), dict(k=q.half()), dict(q=q[..., :60], k=q[..., :60]),
                dict(cos=cos[:3], sin=sin[:3]), dict(sin=None), dict(layout="pairs"), dict(cos=cos[:, :12], sin=sin[:, :12]),
                dict(q_weight=torch.ones(63, device="cuda")), dict(q_weight=torch.ones(64)), dict(cos=cos.cpu(), sin=sin.cpu()),
                dict(out=(q[:, :1], q)), dict(out=(q.transpose(2, 3).contiguous().transpose(2, 3), q))):
        args = dict(q=q, k=q, cos=cos, sin=sin)
        args.update(bad)
        with pytest.raises((ValueError, TypeError)):
            qk_norm_rope(**args)
    with pytest.raises(RuntimeError, match="no backward"):
        qk_norm_rope(q.clone().requires_grad_(), q, cos, sin)
