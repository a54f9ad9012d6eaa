"""Rotary plans on another stream than their own."""

import pytest
import torch

from shellsmith_b200 import paged, rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("append,compiled", [(False, False), (True, False), (True, True)])
def test_plan_dropped_behind_queued_work(cuda, monkeypatch, append, compiled):
    """A plan laid out on one stream, used on another and dropped there at once: its tables'
    memory is not handed out while the call is still queued, and the result is the same."""
    def call(plan):
        if not append:
            return torch.cat([t.flatten() for t in rotary.rotary(q, k, pos, plan)])
        return rotary.rotary_append(q, k, k, pos, plan, pool, slots)

    if not compiled:
        monkeypatch.setattr(rotary, "fast", None)
    q = torch.randn((9, 8, 128), device=cuda).to(torch.bfloat16)
    k = torch.randn((9, 2, 128), device=cuda).to(torch.bfloat16)
    pos = torch.arange(100, 109, dtype=torch.int32, device=cuda)
    pool, slots = paged.new_pool(2, 2, 128, device=cuda), torch.arange(9, device=cuda)
    want = call(rotary.RotaryPlan(128, device=cuda))
    plan = rotary.RotaryPlan(128, device=cuda)
    old = (plan.turns_ptr, plan.axis_ptr)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        out = call(plan)
    del plan
    taken = [torch.empty((n,), dtype=torch.int32, device=cuda) for n in (64, 128) for _ in range(8)]
    assert not set(old) & {t.data_ptr() for t in taken}
    assert not side.query()              # it was still queued
    for t in taken:
        t.fill_(-1)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
