"""fp16 rows whose largest score stands far above many small ones: what the small
ones add up to is kept.

Tolerance: a probability is rounded to 11 bits (2^-11 of itself), or to half a
step of fp16's subnormals, which is at most 2^-36 of the row's largest
probability; scores and sums as in test_gpu_packed_attention (scores off by at
most (D + 4) 2^-24 sum|q k| scale, counted twice, sums by 2^-20); the output is
rounded once (2^-11 of itself, or 2^-25)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gap", [12.0, 17.0, 18.0, 21.0, 26.0])
@pytest.mark.parametrize("lq,lk,hq,hk,d", [(1, 65536, 2, 2, 64), (4, 40000, 8, 2, 128), (13, 30000, 8, 2, 64),
                                           (300, 65536, 2, 2, 64), (200, 30000, 4, 1, 128)])
def test_tails(lq, lk, hq, hk, d, gap):
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    g = torch.Generator("cuda").manual_seed(lq + lk)
    q = 0.05 * torch.randn(1, hq, lq, d, generator=g, device="cuda")
    k = 0.05 * torch.randn(1, hk, lk, d, generator=g, device="cuda")
    v = 0.5 + torch.rand(1, hk, lk, d, generator=g, device="cuda")
    at = torch.randint(0, lk, (hk,), generator=g, device="cuda")
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[0, torch.arange(hk, device="cuda"), at, 0] = gap * d ** 0.5 / 4      # its score is `gap` above the others'
    v[0, torch.arange(hk, device="cuda"), at] = 0.0                        # and it adds nothing itself
    q, k, v = q.half(), k.half(), v.half()
    out = packed_attention(q, k, v, packed_plan([lq], [lk], heads=hq, kv_heads=hk, head_dim=d)).double()
    kk, vv = (x.double().repeat_interleave(hq // hk, 1) for x in (k, v))
    s = q.double() @ kk.transpose(2, 3) * d ** -0.5
    off = (q.double().abs() @ kk.abs().transpose(2, 3)).amax(-1, keepdim=True) * d ** -0.5 * (d + 4) * 2.0 ** -24
    p = s.softmax(-1)
    ref, size = p @ vv, p @ vv.abs()
    bound = ((2.0 ** -11 + 2 * off + 2.0 ** -20) * size + 2.0 ** -36 * p.amax(-1, keepdim=True) * vv.abs().sum(2, keepdim=True)
             + 2.0 ** -11 * ref.abs() + 2.0 ** -25)
    worst = ((out - ref).abs() / bound).max().item()
    assert worst <= 1.01, f"{worst:.3g} times the bound"
