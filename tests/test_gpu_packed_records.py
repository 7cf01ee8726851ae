"""The C entry point of the packed attention with records that point outside
the buffers or the workspace: they are passed over or cut by the kernels'
bounds checks, and nothing beside the outputs is written."""

import pytest
import torch

pytestmark = pytest.mark.gpu

QL, KL, HQ, HK, D = [1, 20, 2, 400, 70, 300], [4000, 2000, 3000, 900, 70, 5000], 8, 2, 64
SENTINEL = 7.0
FIELDS = ("q0", "lq", "k0", "lk", "r0", "kb", "ke", "slot")


class _Call:
    """One batch through the C ABI on buffers with margins."""

    def __init__(self):
        import ctypes
        from comfyui_vc_attention_b200.vc_attention import _native as N, packed_plan
        self.N, self.ctypes = N, ctypes
        g = torch.Generator("cuda").manual_seed(1)
        self.q, self.k, self.v = (torch.randn(n, h, D, generator=g, device="cuda").to(torch.bfloat16)
                                  for n, h in ((sum(QL), HQ), (sum(KL), HK), (sum(KL), HK)))
        self.plan = packed_plan(QL, KL, heads=HQ, kv_heads=HK, head_dim=D, causal=True)
        assert all(len(t) for t in self.plan.tiles) and all(self.plan.work.slots)   # every list, each with split tiles
        self.ws_words = self.plan.workspace_bytes // 4

    def run(self):
        N, c = self.N, self.ctypes
        buf = torch.full((sum(QL) + 64, HQ, D), SENTINEL, device="cuda", dtype=torch.bfloat16)
        ws = torch.full((self.ws_words + 8192,), SENTINEL, device="cuda")
        view = lambda t: N.BHND(t.data_ptr(), 0, t.stride(1), t.stride(0))  # noqa: E731
        out = buf[32:-32]
        args = [view(t) for t in (self.q, self.k, self.v, out)]
        N.check("vcattn_attn_packed", N.lib().vcattn_attn_packed(
            c.byref(args[0]), c.byref(args[1]), c.byref(args[2]), N.DTYPE_BF16, HQ, HK, sum(QL), sum(KL), D,
            c.byref(self.plan.work), 1, D ** -0.5, c.byref(args[3]), ws[4096:].data_ptr(), self.ws_words * 4,
            torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert (buf[:32] == SENTINEL).all() and (buf[-32:] == SENTINEL).all()
        assert (ws[:4096] == SENTINEL).all() and (ws[4096 + self.ws_words:] == SENTINEL).all()
        return out


BAD = [("q0", -1), ("q0", -2 ** 31), ("q0", 2 ** 31 - 1), ("lq", -5), ("lq", 2 ** 31 - 1), ("k0", -1), ("k0", 2 ** 31 - 1),
       ("lk", -3), ("lk", 2 ** 31 - 1), ("r0", -64), ("r0", 2 ** 31 - 1), ("kb", -64), ("ke", 2 ** 31 - 1), ("ke", -9),
       ("slot", 2 ** 30), ("slot", "slots"), ("slot", -7)]


@pytest.mark.parametrize("field,value", BAD)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_tiles(which, field, value):
    call = _Call()
    want = call.run().clone()
    tiles = call.plan.tiles[which]
    split = int((tiles[:, 7] >= 0).nonzero()[0])
    keep = tiles[split].clone()
    if value == "slots":
        value = call.plan.work.slots[which]
    tiles[split, FIELDS.index(field)] = value
    got = call.run()
    same = torch.ones(sum(QL), dtype=torch.bool, device="cuda")
    same[int(keep[0]):int(keep[0] + keep[1])] = False        # the rows of the record's own sequence are its own affair
    assert torch.equal(got[same], want[same])
    tiles[split] = keep
    assert torch.equal(call.run(), want)


@pytest.mark.parametrize("column,value", [(0, -1), (0, 2 ** 31 - 1), (1, -5), (1, 2 ** 31 - 1), (2, -64), (2, 2 ** 31 - 1),
                                          (3, -1), (3, 2 ** 30), (4, -1), (4, 2 ** 30), (4, "more")])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_joins(which, column, value):
    call = _Call()
    want = call.run().clone()
    joins = call.plan.joins[which]
    at = len(joins) - 1
    keep = joins[at].clone()
    if value == "more":                                       # one part past the last
        value = call.plan.work.slots[which] - int(keep[3]) + 1
    joins[at, column] = value
    got = call.run()
    same = torch.ones(sum(QL), dtype=torch.bool, device="cuda")
    same[int(keep[0]):int(keep[0] + keep[1])] = False
    assert torch.equal(got[same], want[same])
