"""The ways into the group-decode operators: the compiled callers, the Python wrappers
behind them and torch.ops.shellcache.* launch the same kernels with the same arguments, so
their results are the same bits; what one refuses, the other refuses with the same error."""

import pytest
import torch

from shellsmith_b200 import _capi, _torch, beam, paged, rotary, torch_ops  # noqa: F401 (registers)

pytestmark = pytest.mark.gpu


@pytest.fixture
def without_fast(monkeypatch):
    def switch():
        for module in (rotary, beam, paged):
            monkeypatch.setattr(module, "fast", None)
    return switch


def _rand(cuda, *shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator(device=cuda).manual_seed(seed),
                       device=cuda).to(dtype)


def _rotary_call(cuda, strided, append, weights):
    q, k, v = (_rand(cuda, 9, h, 128 * 2, seed=h)[..., :128] for h in (8, 2, 3))
    v = v[:, :2]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    plan = rotary.RotaryPlan(128, 64, sections=(12, 10, 10), interleaved=True, device=cuda)
    pos = torch.arange(27, dtype=torch.int32, device=cuda).view(3, 9)
    w = dict(q_weight=_rand(cuda, 128, seed=5), k_weight=_rand(cuda, 128, seed=6)) if weights else {}
    if not append:
        return [*rotary.rotary(q, k, pos, plan, **w)]
    pool = paged.new_pool(4, 2, 128, device=cuda).zero_()
    slots = torch.tensor([5, -1, 17, 63, 0, 1, 2, 3, 40], device=cuda)
    return [rotary.rotary_append(q, k, v, pos, plan, pool, slots, **w), pool]


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_rotary_callers_agree(cuda, without_fast, strided, append, weights):
    assert _torch.fast is not None
    a = _rotary_call(cuda, strided, append, weights)
    without_fast()
    for x, y in zip(a, _rotary_call(cuda, strided, append, weights), strict=True):
        assert torch.equal(x, y)


def _attention_case(cuda):
    pool = _rand(cuda, 64, 2, 2, 16, 128)
    table = torch.randperm(64, generator=torch.Generator().manual_seed(2))[:48].view(4, 12)
    table[1:3, :8] = table[0, :8]
    table = table.to(cuda, torch.int32)
    ctx = torch.tensor([150, 129, 192, 77], dtype=torch.int32, device=cuda)
    groups = [([0, 1, 2], 128)]
    return _rand(cuda, 4, 16, 128, seed=3), pool, table, ctx, groups


@pytest.mark.parametrize("lengths", [False, True])
def test_attention_callers_agree(cuda, without_fast, lengths):
    q, pool, table, ctx, groups = _attention_case(cuda)
    plan = paged.PrefixGroups(groups, 4, 16, 2, 128, device=cuda)
    kw = dict(max_suffix_pages=5, total_suffix_pages=2 + 1 + 4 + 5) if lengths else {}
    lse = [torch.empty(4 * 16, device=cuda) for _ in range(2)]
    a = paged.shared_prefix_attention(q, pool, table, ctx, 0.09, plan, lse_out=lse[0], **kw)
    op = torch.ops.shellcache.shared_prefix_attention(q, pool, table, ctx, 0.09, [0, 1, 2], [3],
                                                      [128], **kw)
    without_fast()
    b = paged.shared_prefix_attention(q, pool, table, ctx, 0.09, plan, lse_out=lse[1], **kw)
    assert torch.equal(a, b) and torch.equal(*lse) and torch.equal(a, op)
    with pytest.raises(ValueError):
        torch.ops.shellcache.shared_prefix_attention(q, pool, table, ctx, 0.09, [0, 1, 2], [2],
                                                     [128])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("finished", [False, True])
def test_beam_callers_agree(cuda, without_fast, dtype, finished):
    logits, scores = _rand(cuda, 3, 4, 5003, dtype=dtype), _rand(cuda, 3, 4, dtype=torch.float32)
    done = torch.tensor([[0, 1, 0, 0], [0, 0, 0, 0], [1, 1, 1, 1]], device=cuda).bool() \
        if finished else None
    a = beam.beam_select(logits, scores, 6, finished=done, pad_token=7)
    op = torch.ops.shellcache.beam_select(logits, scores, 6, done, 7)
    without_fast()
    b = beam.beam_select(logits, scores, 6, finished=done, pad_token=7)
    for x, y, z in zip(a, b, op, strict=True):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_reorder_callers_agree(cuda, without_fast):
    slots = torch.tensor([[3, 9, 0], [7, 4, 5]], dtype=torch.int32, device=cuda)
    parents = torch.tensor([[1, 1, 1], [2, 0, 2]], dtype=torch.int32, device=cuda)
    pools = lambda: [_rand(cuda, 2, 10, 4, 64, dtype=torch.float32), _rand(cuda, 3, 10, 24)]  # noqa: E731
    a, b, c = pools(), pools(), pools()
    new = [beam.reorder_rows(a, slots, parents), torch.ops.shellcache.reorder_rows(c, slots, parents)]
    without_fast()
    new.append(beam.reorder_rows(b, slots, parents))
    assert torch.equal(new[0], new[1]) and torch.equal(new[0], new[2])
    for x, y, z in zip(a, b, c, strict=True):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_rotary_operator_equals_the_call(cuda):
    q, k = _rand(cuda, 6, 8, 128), _rand(cuda, 6, 2, 128, seed=1)
    pos = torch.arange(12, dtype=torch.int32, device=cuda).view(2, 6)
    slots = torch.arange(6, device=cuda)
    a, b = (paged.new_pool(2, 2, 128, device=cuda).zero_() for _ in range(2))
    got = torch.ops.shellcache.rotary_append(q, k, k, pos, a, slots, 64, 1e6, [20, 12], False, None,
                                             _rand(cuda, 128, seed=4))
    plan = rotary.RotaryPlan(128, 64, base=1e6, sections=(20, 12), device=cuda)
    want = rotary.rotary_append(q, k, k, pos, plan, b, slots, k_weight=_rand(cuda, 128, seed=4))
    assert torch.equal(got, want) and torch.equal(a, b)


def test_schema_and_fake_checks(cuda):
    check = lambda op, *args: torch.library.opcheck(  # noqa: E731
        op, args, test_utils=("test_schema", "test_faketensor"))
    ops = torch.ops.shellcache
    q, pool, table, ctx, _ = _attention_case(cuda)
    check(ops.shared_prefix_attention, q, pool, table, ctx, 0.09, [0, 1, 2], [3], [128])
    check(ops.beam_select, _rand(cuda, 2, 3, 999), _rand(cuda, 2, 3, dtype=torch.float32), 4)
    slots = torch.tensor([[3, 9, 0]], dtype=torch.int32, device=cuda)
    parents = torch.tensor([[1, 1, 0]], dtype=torch.int32, device=cuda)
    check(ops.reorder_rows, [_rand(cuda, 2, 10, 64)], slots, parents)
    k = _rand(cuda, 4, 2, 128)
    check(ops.rotary_append, q, k, k, ctx[None], pool, torch.arange(4, device=cuda), 64)


def _refusals(cuda):
    """(error, call): everything the callers have to refuse before a launch."""
    q, pool, table, ctx, groups = _attention_case(cuda)
    plan = paged.PrefixGroups(groups, 4, 16, 2, 128, device=cuda)
    attend = lambda q=q, pool=pool, table=table, ctx=ctx, **kw: (  # noqa: E731
        lambda: paged.shared_prefix_attention(q, pool, table, ctx, 0.1, plan, **kw))
    logits, scores = _rand(cuda, 2, 3, 100), _rand(cuda, 2, 3, dtype=torch.float32)
    select = lambda logits=logits, scores=scores, n=3, **kw: (  # noqa: E731
        lambda: beam.beam_select(logits, scores, n, **kw))
    slots = torch.tensor([[0, 1]], dtype=torch.int32, device=cuda)
    move = lambda pools, s=slots, p=slots: lambda: beam.reorder_rows(pools, s, p)  # noqa: E731
    state = _rand(cuda, 2, 4, 64)
    rp = rotary.RotaryPlan(128, device=cuda)
    k, pos, where = _rand(cuda, 4, 2, 128), ctx[None], torch.arange(4, device=cuda)
    put = lambda q=q, k=k, v=k, pos=pos, pool=pool, where=where, **kw: (  # noqa: E731
        lambda: rotary.rotary_append(q, k, v, pos, rp, pool, where, **kw))
    both = (ValueError, TypeError, _capi.ShellcacheError)
    return [
        (both, attend(q=q.cpu())), (both, attend(q=q.float())), (both, attend(q=q[:3])),
        (both, attend(q=q[..., :64])), (both, attend(table=table.long())),
        (both, attend(table=table[:3])), (both, attend(ctx=ctx.long())), (both, attend(ctx=ctx[:2])),
        (both, attend(pool=pool.float())), (both, attend(pool=pool[..., :64])),
        (both, attend(out=torch.empty(4, 16, 64, device=cuda, dtype=torch.bfloat16))),
        (both, attend(lse_out=torch.empty(4, device=cuda))),
        (both, select(logits=logits.cpu())), (both, select(logits=logits.half())),
        (both, select(logits=logits[0])), (both, select(scores=scores.double())),
        (both, select(scores=scores[:1])), (both, select(n=0)), (both, select(n=65)),
        (both, select(logits=logits[..., ::2])), (both, select(finished=scores)),
        (both, select(finished=torch.zeros(2, 2, dtype=torch.bool, device=cuda))),
        (both, select(logits=logits.expand(2, 3, 100)[:, :1].expand(2, 70, 100),
                      scores=_rand(cuda, 2, 70, dtype=torch.float32))),
        (both, move([state] * 5)), (both, move([state.cpu()])), (both, move([state[:, ::2]])),
        (both, move([state], slots.long())), (both, move([state], slots, slots[:, :1])),
        (both, move([state, _rand(cuda, 2, 5, 64)])), (both, move([_rand(cuda, 2, 4, 3)])),
        (both, put(q=q.cpu())), (both, put(q=q.float())), (both, put(k=k[:3])),
        (both, put(v=k[:, :1])), (both, put(pos=pos.long())), (both, put(pos=pos[:, :3])),
        (both, put(pos=pos.expand(2, 4))), (both, put(where=where.int())),
        (both, put(where=where[:2])), (both, put(pool=pool[..., :64])),
        (both, put(pool=pool[:, :1])), (both, put(q_weight=_rand(cuda, 64))),
    ]


def test_both_ways_refuse_the_same(cuda, without_fast):
    def errors():
        out = []
        for i, (kinds, call) in enumerate(_refusals(cuda)):
            with pytest.raises(kinds) as err:
                call()
                pytest.fail(f"call {i} was not refused")
            out.append((type(err.value), str(err.value)))
        return out
    compiled = errors()
    without_fast()
    assert compiled == errors()
    torch.cuda.synchronize()
