"""Shared-prefix decode attention (paged.shared_prefix_attention) at its edges: short tails
over many units of work, infinities in the cache, long sequences without a group. Cases, the
64-bit reference and the bars are those of the operator's own tests."""

import numpy as np
import pytest
import torch
from test_shared_prefix_gpu import _case, _check, _expect

from shellsmith_b200 import _capi, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,D", [(4, 2, 256), (4, 4, 128)])
@pytest.mark.parametrize("longest", [15, 17, 33])
def test_many_short_tails(cuda, hq, hkv, D, longest):
    """Several units a warp, of one to three pages, most ending inside a page: the rows past
    a context are cleared in shared memory, and the next page lands on them."""
    groups = [(700, 32), (500, 16)]
    tails = [1 + (5 * i) % longest for i in range(1200)]
    case = _case(cuda, groups, tails, hq, hkv, D, seed=longest)
    for _ in range(3):
        _check(cuda, case)


def _prepared(cuda, case, ws, scale=0.0625):
    """The call of a case with everything on the device before it: nothing in it waits."""
    q, pool, table, ctx, plan = case
    groups = paged.PrefixGroups(plan, q.shape[0], q.shape[1], pool.shape[1], q.shape[2], device=cuda)
    t, c = torch.from_numpy(table).to(cuda), torch.from_numpy(ctx.astype(np.int32)).to(cuda)
    return lambda: paged.shared_prefix_attention(q, pool, t, c, scale, groups, workspace=ws)


def _matches(out, case, scale=0.0625):
    q, pool, table, ctx, _ = case
    want, _, mass = _expect(q, pool, table, ctx, scale)
    tol = (2.0 ** -8 + 3e-4) * mass + 2.0 ** -8 * 1.01 * np.abs(want) + 1e-6
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all()


def test_workspace_memory_outlives_the_work_on_it(cuda):
    """A workspace from one stream grows on another: its old memory is not handed out on the
    first while the second still has work on it."""
    small = _case(cuda, [(3, 160)], [1, 9, 30], 16, 2, 256, seed=1)
    large = _case(cuda, [(9, 1600)], [1 + 31 * i for i in range(9)], 16, 2, 256, seed=2)
    ws = paged.SharedPrefixWorkspace(cuda)
    one, two = _prepared(cuda, small, ws), _prepared(cuda, large, ws)
    one()
    floats, old = ws._floats, ws._buffer.data_ptr()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)   # about 0.1 s: the call below is still queued
        a = one()
        b = two()
    assert ws._floats > floats
    fresh = torch.empty(floats, dtype=torch.float32, device=cuda)
    assert fresh.data_ptr() != old
    assert not side.query()              # it was still queued
    fresh.fill_(float("nan"))
    torch.cuda.synchronize()
    _matches(a, small)
    _matches(b, large)


def test_workspace_of_a_captured_call(cuda):
    """A graph keeps the memory that it was captured with when the workspace grows."""
    small = _case(cuda, [(3, 160)], [1, 9, 30], 16, 2, 256, seed=1)
    large = _case(cuda, [(9, 1600)], [1 + 31 * i for i in range(9)], 16, 2, 256, seed=2)
    ws = paged.SharedPrefixWorkspace(cuda)
    one, two = _prepared(cuda, small, ws), _prepared(cuda, large, ws)
    one()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one()
    floats, old = ws._floats, ws._buffer.data_ptr()
    b = two()
    torch.cuda.synchronize()
    taken = [torch.zeros(floats, device=cuda) for _ in range(4)]
    assert old not in [t.data_ptr() for t in taken]
    graph.replay()
    torch.cuda.synchronize()
    assert not any(t.any() for t in taken)
    _matches(out, small)
    _matches(b, large)


def test_calls_back_to_back_on_one_workspace(cuda):
    """Calls of different shapes, contexts and counters queued on a side stream with nothing
    between them: each one's first kernel starts while the last of the one before ends, on
    the same parts."""
    cases = [_case(cuda, [(8, 1600)], [1 + 9 * i for i in range(8)], 16, 2, 256, seed=9),
             _case(cuda, [(5, 48), (40, 320)], [1 + (7 * i) % 90 for i in range(45)], 24, 8, 128, seed=3),
             _case(cuda, [(3, 5000)], [2000, 1, 40], 8, 8, 64, seed=4),
             _case(cuda, [(2, 160)], [-100, None], 16, 2, 256, seed=5)]
    ws = paged.SharedPrefixWorkspace(cuda)
    calls = [_prepared(cuda, c, ws) for c in cases]
    for call in calls:  # grown to its size, kernels loaded
        call()
    torch.cuda.synchronize()
    order = [0, 1, 2, 3, 3, 2, 0, 0, 1, 3, 1, 2, 0, 3, 2, 1] * 4
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the queue fills before the first one runs
        outs = [calls[i]() for i in order]
    side.synchronize()
    _capi.check_device(side.cuda_stream)
    first = {}
    for i, out in zip(order, outs):
        if i not in first:
            first[i] = out
            _matches(out, cases[i])
        assert torch.equal(out, first[i])


def _decode(cuda, case, scale, sms=None):
    q, pool, table, ctx, plan = case
    groups = paged.PrefixGroups(plan, q.shape[0], q.shape[1], pool.shape[1], q.shape[2], device=cuda,
                                sms=sms)
    t, c = torch.from_numpy(table).to(cuda), torch.from_numpy(ctx.astype(np.int32)).to(cuda)
    out = paged.shared_prefix_attention(q, pool, t, c, scale, groups)
    _capi.check_device()
    return out, paged.paged_decode_attention(q, pool, t, c, scale)


@pytest.mark.parametrize("hq,hkv,D", [(16, 2, 256), (24, 8, 128), (8, 8, 64), (64, 1, 64)])
@pytest.mark.parametrize("sms", [1, 148])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_pages_past_a_members_context_do_not_reach_it(cuda, hq, hkv, D, sms, value):
    """Members whose contexts end inside the shared pages, which hold infinities or NaN past
    them, as K or as V: their rows are those of the finite tokens that they attend to."""
    pages = 40
    tails = [5, -1, -16, -100, -300, None, 0, -17, -639 + 16]
    case = _case(cuda, [(len(tails), pages * 16)], tails, hq, hkv, D, seed=7)
    q, pool, table, ctx, _ = case
    shared = torch.from_numpy(table[0, :pages].astype(np.int64)).to(cuda)
    for last, which in ((20, 1), (1, 1), (39, 1), (30, 0), (7, 0)):
        bad = pool.clone()
        bad[shared[last:], :, which] = value
        rows = [i for i, n in enumerate(ctx) if n <= 16 * last]
        assert rows and len(rows) < len(tails)
        now = (q, bad, table, ctx, case[4])
        out, plain = _decode(cuda, now, 0.06, sms)
        want, _, mass = _expect(q, pool, table, ctx, 0.06)
        tol = (2.0 ** -8 + 3e-4) * mass + 2.0 ** -8 * 1.01 * np.abs(want) + 1e-6
        got = out.double().cpu().numpy()
        assert np.isfinite(got[rows]).all() and torch.isfinite(plain[rows]).all()
        assert (np.abs(got - want)[rows] <= tol[rows]).all()


@pytest.mark.parametrize("pages", [37, 38, 39, 40])
@pytest.mark.parametrize("D", [64, 256])
def test_an_infinite_value_stays_infinite(cuda, pages, D):
    """V of +Inf in one column of the last shared page, inside a tile of the kernel or not:
    that column is +Inf, as p > 0 there, and the others are what they were."""
    case = _case(cuda, [(3, pages * 16)], [1, 30, 17], 8, 2, D, seed=8)
    q, pool, table, ctx, _ = case
    want, plain = _decode(cuda, case, 0.05)
    bad = pool.clone()
    token, col = 5, 24                                     # stored at chunk 3 ^ 5 of the row
    bad[int(table[0, pages - 1]), :, 1, token, ((col // 8) ^ token) * 8 + col % 8] = float("inf")
    out, plain = _decode(cuda, (q, bad, table, ctx, case[4]), 0.05)
    assert torch.isposinf(out[..., col]).all() and torch.isposinf(plain[..., col]).all()
    rest = torch.arange(D, device=cuda) != col
    assert torch.equal(out[..., rest], want[..., rest])


@pytest.mark.parametrize("hq,hkv,D", [(16, 2, 256), (12, 1, 128), (8, 8, 64)])
def test_tokens_with_scores_of_minus_infinity_weigh_nothing(cuda, hq, hkv, D):
    """Keys of -Inf against a positive entry of q: whole pages of them, first in the prefix,
    first in a sequence's own pages (and in a unit of those by themselves), and single ones."""
    case = _case(cuda, [(3, 320)], [200, 17, 90], hq, hkv, D, seed=11, single=[60])
    q, pool, table, ctx, _ = case
    q[..., 0] = q[..., 0].abs() + 1
    def kill(b, tokens):
        for t in tokens:
            page, row = int(table[b, t // 16]), t % 16
            pool[page, :, 0, row, 8 * (row & 7)] = -float("inf")  # column 0 of its row
    kill(0, range(0, 33))                # two pages of the prefix and a token
    kill(0, range(320, 320 + 64))        # the first unit of row 0's own pages
    kill(1, range(320, 336))             # its first own page, one token left
    kill(2, [320, 350, 409])
    kill(3, range(0, 16))
    _check(cuda, case)
    for splits in (1, 2, 8):
        _check(cuda, case, pages_per_split=splits)


@pytest.mark.parametrize("hq,hkv,D", [(16, 2, 256), (6, 1, 128), (8, 8, 64)])
@pytest.mark.parametrize("pages_per_split", [31, 32, 33, 64, 100])
def test_units_of_more_pages_than_a_warp_has_lanes(cuda, hq, hkv, D, pages_per_split):
    case = _case(cuda, [(2, 48), (2, 160)], [40 * 16, 1, 33 * 16, 66 * 16 + 5], hq, hkv, D, seed=13,
                 single=[130 * 16 - 3, 20])
    _check(cuda, case, pages_per_split=pages_per_split)


@pytest.mark.parametrize("tokens,hint", [(70_000, True), (70_000, False), (290_000, True)])
def test_a_long_sequence_beside_a_group(cuda, tokens, hint):
    """One kv head: more parts of 4, 8 or 16 pages than the entry point takes, so longer ones."""
    case = _case(cuda, [(2, 64)], [5, 30], 4, 1, 64, seed=14, single=[tokens])
    _check(cuda, case, hint=hint)


@pytest.mark.parametrize("compiled", [False, True])
def test_groups_dropped_behind_queued_work(cuda, monkeypatch, compiled):
    """Groups laid out on one stream, used on another and dropped there at once: their tables'
    memory is not handed out while the call is still queued."""
    case = _case(cuda, [(3, 160), (4, 320)], [1, 9, 30, 4, 5, 6, 70], 16, 2, 256, seed=1)
    q, pool, table, ctx, plan = case
    t, c = torch.from_numpy(table).to(cuda), torch.from_numpy(ctx.astype(np.int32)).to(cuda)
    ws = paged.SharedPrefixWorkspace(cuda)
    _prepared(cuda, case, ws)()          # grown to its size
    if not compiled:
        monkeypatch.setattr(paged, "fast", None)
    groups = paged.PrefixGroups(plan, 7, 16, 2, 256, device=cuda)
    old, size = groups.tiles_ptr, groups.tiles.untyped_storage().nbytes()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        out = paged.shared_prefix_attention(q, pool, t, c, 0.0625, groups, workspace=ws)
    del groups
    taken = [torch.empty((size // 4,), dtype=torch.int32, device=cuda) for _ in range(8)]
    assert old not in [x.data_ptr() for x in taken]
    assert not side.query()
    for x in taken:
        x.fill_(-1)
    torch.cuda.synchronize()
    _capi.check_device()
    _matches(out, case)
