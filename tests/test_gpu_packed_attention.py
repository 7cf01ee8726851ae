"""packed_attention against softmax in 64 bits, sequence by sequence.

Tolerance: P is rounded to the input type (half a unit u = 2^-8 bf16, 2^-11
fp16, relative to each probability), so the row is off by at most
u * sum p|v|; the fp32 scores are off by at most (D + 4) 2^-24 sum|q k| scale,
which moves numerator and denominator by that relative amount each; and the
output is rounded once (u |o|, 2^-25 below fp16's normal range).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _inputs(ql, kl, hq, hk, d, dtype, seed=0, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: torch.randn(n, h, d, generator=g, device="cuda")  # noqa: E731
    q, k, v = r(sum(ql), hq), r(sum(kl), hk) + offset * r(1, hk), r(sum(kl), hk)
    return tuple(x.to(dtype).transpose(0, 1).unsqueeze(0) for x in (q, k, v))


def _check(out, q, k, v, ql, kl, causal, scale=None):
    d, rep = q.shape[-1], q.shape[1] // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    u = HALF_UNIT[q.dtype]
    assert out.shape == q.shape and out.dtype == q.dtype
    q0 = k0 = 0
    for a, b in zip(ql, kl):
        qq = q[0, :, q0:q0 + a].double()
        kk = k[0, :, k0:k0 + b].double().repeat_interleave(rep, 0)
        vv = v[0, :, k0:k0 + b].double().repeat_interleave(rep, 0)
        got = out[0, :, q0:q0 + a].double()
        s = qq @ kk.transpose(1, 2) * scale
        off = (qq.abs() @ kk.abs().transpose(1, 2) * scale).amax(-1, keepdim=True) * (d + 4) * 2.0 ** -24 \
            if b else torch.zeros(q.shape[1], a, 1, device="cuda")
        if causal:
            hide = torch.arange(b, device="cuda") > torch.arange(a, device="cuda")[:, None] + b - a
            s = s.masked_fill(hide, -math.inf)
        live = (s > -math.inf).any(-1, keepdim=True) if b else torch.zeros_like(off, dtype=torch.bool)
        p = torch.softmax(s, -1).nan_to_num(0.0) if b else s
        ref, size = p @ vv, p @ vv.abs()
        bound = (u + 2 * off + 2.0 ** -20) * size + u * ref.abs() + 2.0 ** -25
        bad = (got - ref).abs() > 1.01 * bound
        assert not bad.any(), f"sequence {a} x {b}: {int(bad.sum())} of {bad.numel()} outside the bound, " \
                              f"{((got - ref).abs() / bound).max().item():.3g} times it"
        assert (got[~live.expand_as(got)] == 0).all()
        q0, k0 = q0 + a, k0 + b


def _run(ql, kl, hq, hk, d, dtype, causal, **kw):
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v = _inputs(ql, kl, hq, hk, d, dtype)
    plan = packed_plan(ql, kl, heads=hq, kv_heads=hk, head_dim=d, causal=causal)
    _check(packed_attention(q, k, v, plan, **kw), q, k, v, ql, kl, causal, kw.get("scale"))


LENGTHS = [
    ([1], [1]), ([1], [64]), ([1], [65]), ([64], [64]), ([63], [129]), ([65], [63]), ([128], [128]), ([257], [257]),
    ([1, 77, 0, 200, 333], [1, 77, 0, 200, 333]), ([5, 0, 3], [0, 9, 2]), ([130, 1, 17], [1, 1000, 400]),
    ([300], [20]), ([300, 2, 30], [0, 0, 0]), ([700, 64, 90, 513, 300], [20, 700, 64, 1100, 300]), ([1, 1, 1, 1], [2500, 1, 129, 640]), ([129, 255, 256], [511, 255, 1024]), ([700], [1500])]


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 64),
                                     (torch.float16, 128)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ql,kl", LENGTHS, ids=lambda x: "-".join(map(str, x)))
def test_lengths(ql, kl, causal, dtype, d):
    _run(ql, kl, 4, 2, d, dtype, causal)


@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 6), (32, 8), (40, 8), (7, 1), (16, 1), (96, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_head_groups(hq, hk, causal):
    _run([1, 200, 33], [300, 200, 90], hq, hk, 128, torch.bfloat16, causal)


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_scale(scale):
    _run([150], [170], 2, 2, 64, torch.float16, True, scale=scale)


def test_long_history_of_single_tokens():
    _run([1] * 6, [16384, 3, 4097, 8192, 1, 12000], 8, 2, 128, torch.bfloat16, True)


def test_long_sequence():
    _run([2048, 1024], [4096, 1024], 2, 1, 128, torch.bfloat16, True)
    _run([3000], [2990], 2, 2, 64, torch.float16, False)


def test_many_items_per_sm():
    """More (tile, head) pairs than SMs, of unlike lengths, so that every CTA works through several."""
    _run([900, 64, 300, 1, 520, 0, 257], [1200, 64, 10, 300, 520, 5, 900], 56, 56, 64, torch.float16, True)
    _run([1030, 256, 70], [1030, 2000, 1], 40, 8, 128, torch.bfloat16, False)


def test_layouts_out_and_neighbours():
    """(H, T, D) and (T, H, D) buffers, views of a fused projection, a given output."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    ql, h, d = [70, 3, 129], 4, 64
    t = sum(ql)
    qkv = torch.randn(t, 3 * h, d, device="cuda").to(torch.bfloat16)
    q, k, v = (qkv[:, i * h:(i + 1) * h].transpose(0, 1).unsqueeze(0) for i in range(3))
    plan = packed_plan(ql, heads=h, head_dim=d)
    out = packed_attention(q, k, v, plan)
    _check(out, q, k, v, ql, ql, False)
    assert out.transpose(1, 2).is_contiguous()
    again = packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), plan)
    assert torch.equal(again, out) and again.is_contiguous()
    buf = torch.full((t + 2, h, d), 5.0, device="cuda", dtype=torch.bfloat16)
    view = buf[1:t + 1].transpose(0, 1).unsqueeze(0)
    assert packed_attention(q, k, v, plan, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, out) and (buf[0] == 5).all() and (buf[-1] == 5).all()
    odd = torch.randn(1, h, t, 2 * d + 1, device="cuda").to(torch.bfloat16)[..., 1:d + 1]   # copied: rows not aligned
    _check(packed_attention(odd, k, v, plan), odd, k, v, ql, ql, False)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_non_finite_neighbours_and_keys(d, causal):
    """Sequences do not see each other's infinities and NaN, whichever tile they share."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    ql, kl, hq, hk = [40, 150, 30, 300], [40, 200, 30, 300], 2, 1
    q, k, v = _inputs(ql, kl, hq, hk, d, torch.bfloat16)
    plan = packed_plan(ql, kl, heads=hq, kv_heads=hk, head_dim=d, causal=causal)
    want = packed_attention(q, k, v, plan)
    for value in (float("nan"), float("inf")):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        k2[:, :, 40:240], v2[:, :, 40:240], q2[:, :, 40:190] = value, value, value
        got = packed_attention(q2, k2, v2, plan)
        for a, b in ((0, 40), (190, 520)):
            assert torch.equal(got[:, :, a:b], want[:, :, a:b])
        assert got[:, :, 40:190].isnan().all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk,heads", [(1, 400, 2), (100, 100, 2), (300, 300, 2), (200, 500, 2), (400, 400, 200)])
def test_non_finite_keys_behind_the_causal_mask(lq, lk, heads, d):
    """Rows before a key that is infinite or NaN (in k, v or both) do not see it."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v = _inputs([lq], [lk], heads, heads // 2, d, torch.bfloat16)
    plan = packed_plan([lq], [lk], heads=heads, kv_heads=heads // 2, head_dim=d, causal=True)
    want = packed_attention(q, k, v, plan)
    key = lk - max(1, lq // 3)           # the rows from lq - max(1, lq // 3) on see it
    first = lq - max(1, lq // 3)
    for value in (float("nan"), float("inf"), -float("inf")):
        for which in ("k", "v"):
            k2, v2 = k.clone(), v.clone()
            (k2 if which == "k" else v2)[:, :, key] = value
            got = packed_attention(q, k2, v2, plan)
            assert torch.equal(got[:, :, :first], want[:, :, :first]), (value, which)
            if which == "v" and value != value:
                assert got[:, :, first:].isnan().all()


def test_extreme_scores():
    """Scores of +-80 (one key takes all) and equal scores."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v = _inputs([50], [300], 2, 2, 64, torch.float16)
    plan = packed_plan([50], [300], heads=2, head_dim=64)
    _check(packed_attention(8 * q, 8 * k, v, plan), 8 * q, 8 * k, v, [50], [300], False)
    _check(packed_attention(0 * q, k, v, plan), 0 * q, k, v, [50], [300], False)
    _check(packed_attention(-8 * q, 8 * k, v, plan), -8 * q, 8 * k, v, [50], [300], False)


def test_repeated_calls_give_the_same_bits_and_streams():
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    for ql, kl in (([1] * 5, [3000, 5, 700, 8000, 64]), ([500, 30], [500, 900])):
        q, k, v = _inputs(ql, kl, 8, 2, 128, torch.bfloat16)
        plan = packed_plan(ql, kl, heads=8, kv_heads=2, head_dim=128, causal=True)
        first = packed_attention(q, k, v, plan)
        for _ in range(3):
            assert torch.equal(packed_attention(q, k, v, plan), first)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = packed_attention(q, k, v, plan)
        s.synchronize()
        assert torch.equal(got, first)


def test_offsets_past_32_bits():
    """Rows whose element offset is beyond 2^31 (a strided view of a 10 GB buffer)."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    n, d, h = 200, 64, 2
    buf = torch.zeros(n, 24 * 2 ** 20, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(n, 3 * h * d, device="cuda").to(torch.bfloat16)
    buf[:, :3 * h * d] = x
    views = [buf[:, i * h * d:(i + 1) * h * d].view(n, h, d).transpose(0, 1).unsqueeze(0) for i in range(3)]
    assert views[0].stride(2) * (n - 1) > 2 ** 31
    plan = packed_plan([n], heads=h, head_dim=d, causal=True)
    _check(packed_attention(*views, plan), *views, [n], [n], True)


def test_no_wait_ran_out():
    """The tcgen05 kernels' status words after the calls above (and a few more)."""
    import ctypes
    from comfyui_vc_attention_b200.vc_attention import _native as N
    _run([700, 3], [1500, 40], 4, 2, 128, torch.bfloat16, True)
    c = [ctypes.c_int(-1) for _ in range(3)]
    N.check("vcattn_attn_status", N.lib().vcattn_attn_status(*(ctypes.byref(x) for x in c), 0))
    assert c[0].value == 0, [x.value for x in c]


def test_broadcast_keys_and_overlapping_output():
    """Keys expanded over the heads (stride 0) are copied; an expanded output is refused."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v = _inputs([70], [90], 4, 1, 64, torch.float16)
    plan = packed_plan([70], [90], heads=4, kv_heads=4, head_dim=64)
    ke, ve = k.expand(1, 4, 90, 64), v.expand(1, 4, 90, 64)
    _check(packed_attention(q, ke, ve, plan), q, ke, ve, [70], [90], False)
    with pytest.raises(ValueError):
        packed_attention(q, ke, ve, plan, out=q[:, :1].expand(1, 4, 70, 64))


def test_refusals():
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v = _inputs([8], [9], 4, 2, 64, torch.bfloat16)
    plan = packed_plan([8], [9], heads=4, kv_heads=2, head_dim=64)
    for bad in (lambda: packed_attention(q[:, :3], k, v, plan), lambda: packed_attention(q, k[:, :, :8], v, plan),
                lambda: packed_attention(q, k, v[:, :, :8], plan), lambda: packed_attention(q.half(), k, v, plan),
                lambda: packed_attention(q.float(), k.float(), v.float(), plan),
                lambda: packed_attention(q, k, v, plan, scale=0.0), lambda: packed_attention(q, k, v, plan, scale=-1.0),
                lambda: packed_attention(q, k, v, plan, scale=float("nan")),
                lambda: packed_attention(q, k, v, plan, out=q.float()), lambda: packed_attention(q[0], k, v, plan)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        packed_attention(q.cpu(), k, v, plan)
    with pytest.raises(RuntimeError, match="no backward"):
        packed_attention(q.clone().requires_grad_(), k, v, plan)
