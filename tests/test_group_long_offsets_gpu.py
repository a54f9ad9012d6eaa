"""Group-decode operators on tensors whose offsets pass 32 bits (elements or bytes): the far
end is read and written, and nothing else is.

Bars: K/V and states are bit copies; attention and scores as in the operators' own tests
(P and the result rounded to bf16: 2^-8 of sum p |v| and of the result; scores 2e-4).
"""

import math

import pytest
import torch

from shellsmith_b200 import _capi, beam, paged, rotary

pytestmark = pytest.mark.gpu
P, HKV, D = 16, 2, 256
PAGES = (1 << 31) // (HKV * 2 * P * D) + 64  # elements past 2^31, bytes past 2^32


@pytest.fixture(scope="module")
def far_pool():
    pool = paged.new_pool(PAGES, HKV, D, device="cuda").zero_()
    yield pool


def test_rotary_append_and_attention_at_the_far_end(cuda, far_pool):
    pages = torch.arange(PAGES - 12, PAGES).tolist()
    shared, own = pages[:4], [pages[4:7], pages[7:12]]
    ctx = [4 * P + 40, 4 * P + 65]
    table = torch.zeros((2, 9), dtype=torch.int32)
    for b in range(2):
        row = shared + own[b]
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    where = [(0, t) for t in range(4 * P)] + [(b, t) for b in range(2) for t in range(4 * P, ctx[b])]
    slots = torch.tensor([int(table[b, t // P]) * P + t % P for b, t in where], device=cuda)
    n = len(where)
    gen = torch.Generator(device=cuda).manual_seed(1)
    k, v = (torch.randn((n, HKV, D), generator=gen, device=cuda).to(torch.bfloat16) for _ in "kv")
    plan = rotary.RotaryPlan(D, 64, device=cuda)
    zero = torch.zeros((1, n), dtype=torch.int32, device=cuda)  # position 0 turns nothing
    q0 = torch.zeros((n, 1, D), dtype=torch.bfloat16, device=cuda)
    rotary.rotary_append(q0, k, v, zero, plan, far_pool, slots)
    kk, vv = paged.kv_gather(far_pool, slots)
    assert torch.equal(kk, k) and torch.equal(vv, v)
    assert not far_pool[:PAGES - 12].any()
    q = torch.randn((2, 16, D), generator=gen, device=cuda).to(torch.bfloat16)
    groups = paged.PrefixGroups([([0, 1], 4 * P)], 2, 16, HKV, D, device=cuda)
    scale = 1 / math.sqrt(D)
    got = paged.shared_prefix_attention(q, far_pool, table.to(cuda),
                                        torch.tensor(ctx, dtype=torch.int32, device=cuda), scale,
                                        groups).double()
    _capi.check_device()
    for b in range(2):
        rows = [i for i, (o, t) in enumerate(where) if t < 4 * P or o == b]
        kd, vd = (x[rows].double().repeat_interleave(8, 1) for x in (k, v))
        p = torch.softmax(scale * torch.einsum("hd,lhd->hl", q[b].double(), kd), -1)
        want = torch.einsum("hl,lhd->hd", p, vd)
        mass = torch.einsum("hl,lhd->hd", p, vd.abs())
        tol = (2.0 ** -8 + 3e-4) * mass + 2.0 ** -8 * 1.01 * want.abs() + 1e-6
        assert ((got[b] - want).abs() <= tol).all()


def test_beam_select_of_rows_past_32_bits(cuda):
    G, K, V, n = 140, 16, 1_000_003, 5   # 2.24e9 logits
    logits = torch.empty((G, K, V), dtype=torch.bfloat16, device=cuda)
    for g in range(G):
        logits[g].normal_()
    scores = torch.randn((G, K), device=cuda)
    best, parents, tokens = beam.beam_select(logits, scores, n)
    for g in (0, G - 1):
        # One row at a time keeps the fp64 copy small.
        full = torch.stack([scores[g, k].double() + torch.log_softmax(logits[g, k].double(), -1)
                            for k in range(K)])
        at = parents[g].long() * V + tokens[g].long()
        assert len(set(at.tolist())) == n
        top = full.view(-1).topk(n).values
        assert (best[g].double() - top).abs().max() <= 2e-4
        assert (full.view(-1)[at] - best[g].double()).abs().max() <= 2e-4


def test_reorder_rows_past_32_bits(cuda):
    layers, rows = 2, 1100               # rows of 2 MiB: 4.6 GB
    pool = torch.zeros((layers, rows, 32 * 128 * 128), device=cuda)
    mark = torch.arange(rows, device=cuda, dtype=torch.float32)
    pool[:, :, 0] = mark
    pool[:, :, -1] = mark + 0.5
    slots = torch.tensor([[rows - 1, rows - 2, 3]], dtype=torch.int32, device=cuda)
    parents = torch.tensor([[0, 0, 0]], dtype=torch.int32, device=cuda)
    new = beam.reorder_rows([pool], slots, parents)
    assert new.tolist() == [[rows - 1, rows - 2, 3]]
    want = mark.clone()
    want[rows - 2] = want[3] = rows - 1
    assert (pool[:, :, 0] == want).all() and (pool[:, :, -1] == want + 0.5).all()
    assert not pool[:, :, 1:-1].any()
