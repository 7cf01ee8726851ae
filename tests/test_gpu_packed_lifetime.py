"""The records of a plan outlive the plan while work that reads them is not done."""

import gc
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

QL, KL = [130, 1, 20, 70, 300], [130, 3000, 500, 70, 300]


def _case():
    from comfyui_vc_attention_b200.vc_attention import packed_plan
    g = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(1, h, n, 128, generator=g, device="cuda").to(torch.bfloat16)
               for h, n in ((8, sum(QL)), (2, sum(KL)), (2, sum(KL))))
    return q, k, v, packed_plan(QL, KL, heads=8, kv_heads=2, head_dim=128, causal=True)


def _span(plan):
    t = next(t for t in plan.tiles if len(t))
    s = t.untyped_storage()
    return s.data_ptr(), s.nbytes()


def _active():
    """Bytes that are in use, or still wait for a stream."""
    return torch.cuda.memory_stats()["active_bytes.all.current"]


def _handed_out(span, stream=None):
    """Is any of this memory in 64 new buffers of its size?  (They are not written.)"""
    with torch.cuda.stream(stream or torch.cuda.current_stream()):
        taken = [torch.empty(span[1], dtype=torch.uint8, device="cuda") for _ in range(64)]
    return any(t.data_ptr() < span[0] + span[1] and span[0] < t.data_ptr() + t.numel() for t in taken)


def test_plan_dropped_while_another_stream_has_not_run_the_call():
    from comfyui_vc_attention_b200.vc_attention import packed_attention
    q, k, v, plan = _case()
    want = packed_attention(q, k, v, plan)
    side, span = torch.cuda.Stream(), _span(plan)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)        # about 0.5 s
        got = packed_attention(q, k, v, plan)
    del plan
    gc.collect()
    assert not _handed_out(span) and not side.query()
    held = _active()
    side.synchronize()
    torch.empty(1, device="cuda")               # (the allocator looks at its events when asked for memory)
    assert _active() <= held - span[1]
    assert torch.equal(got, want)


def test_plan_dropped_after_a_capture():
    from comfyui_vc_attention_b200.vc_attention import packed_attention, packed_plan
    q, k, v, plan = _case()
    want = packed_attention(q, k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        packed_attention(q, k, v, plan)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(q, k, v, plan)
        again = packed_attention(q, k, v, plan)
    span = _span(plan)
    del plan
    gc.collect()
    torch.cuda.synchronize()
    assert not _handed_out(span) and not _handed_out(span, side)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(again, want)
    # the graph's end lets them go, at a later call
    torch.cuda.synchronize()
    del out, again
    held = _active()
    graph.reset()
    del graph
    gc.collect()
    for _ in range(50):
        torch.cuda.synchronize()
        time.sleep(0.02)
        packed_plan([1], heads=1, head_dim=64)
        torch.empty(1, device="cuda")
        if _active() <= held - span[1]:
            break
    assert _active() <= held - span[1]
