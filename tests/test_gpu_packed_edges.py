"""packed_attention at ragged tile ends: warps whose lanes part (rows past the
sequence's end, rows that see different numbers of infinite or NaN keys)
between the loads of their output row from tensor memory."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [(267, 267), (129, 700), (385, 1030), (45, 45)])
def test_rows_that_see_different_numbers_of_infinite_keys(lq, lk, d):
    """Key x of channel c is infinite: every row that sees it gives infinity there,
    the other rows and channels keep their bits."""
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    heads = 24
    g = torch.Generator("cuda").manual_seed(lq)
    q, k, v = (torch.randn(1, heads, n, d, generator=g, device="cuda").to(torch.bfloat16) for n in (lq, lk, lk))
    plan = packed_plan([lq], [lk], heads=heads, head_dim=d, causal=True)
    want = packed_attention(q, k, v, plan)
    v2 = v.clone()
    first = {}                                    # channel -> first row that sees its infinite key
    for i, row in enumerate(range(1, lq, 3)):     # rows of every warp, in changing channel groups
        c = (37 * i) % d
        if c not in first:
            first[c] = row
            v2[:, :, row + lk - lq, c] = float("inf")
    got = packed_attention(q, k, v2, plan)
    rows = torch.arange(lq, device="cuda")
    hit = torch.zeros(lq, d, dtype=torch.bool, device="cuda")
    for c, row in first.items():
        hit[:, c] = rows >= row
    hit = hit.expand(1, heads, lq, d)
    assert (got[hit] == float("inf")).all()
    assert torch.equal(got[~hit], want[~hit])
