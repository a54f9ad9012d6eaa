"""Host logic of group decode (no GPU): plans, page bookkeeping, operator registration."""

import ctypes

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from shellsmith_b200 import _capi, beam, paged, rotary, torch_ops
from shellsmith_b200.block_manager import BlockManager


def test_axis_of_pairs():
    assert rotary.axis_of_pairs([4], False) == [0] * 4
    assert rotary.axis_of_pairs([2, 1, 1], False) == [0, 0, 1, 2]
    assert rotary.axis_of_pairs([3, 2, 1], True) == [0, 1, 2, 0, 1, 0]
    assert rotary.axis_of_pairs([4, 1, 1], True) == [0, 1, 2, 0, 0, 0]
    for sections in ([11, 11, 10], [24, 20, 20], [1, 1, 14]):
        axes = rotary.axis_of_pairs(sections, True)
        assert len(axes) == sum(sections) and set(axes) <= set(range(len(sections)))


def test_rotary_plan_values_and_refusals():
    plan = rotary.RotaryPlan(128, 32, base=1e4, sections=(8, 4, 4), device="cpu")
    want = 1e4 ** (-np.arange(16) / 16) / (2 * np.pi)
    assert np.allclose(plan.turns.numpy(), want, rtol=1e-15) and plan.axes == 3
    assert plan.axis.tolist() == [0] * 8 + [1] * 4 + [2] * 4
    for bad in (dict(head_dim=96), dict(head_dim=64, rotary_dim=72),
                dict(head_dim=64, rotary_dim=8), dict(head_dim=64, rotary_dim=128),
                dict(head_dim=64, sections=(1, 2)), dict(head_dim=64, sections=(40, -8)),
                dict(head_dim=64, inv_freq=[1.0])):
        with pytest.raises(ValueError):
            rotary.RotaryPlan(device="cpu", **bad)


@pytest.mark.parametrize("parents,new,copies", [
    ([0, 1, 2, 3], [10, 11, 12, 13], []),
    ([3, 2, 1, 0], [13, 12, 11, 10], []),
    ([1, 1, 1, 1], [11, 10, 12, 13], [(11, 10), (11, 12), (11, 13)]),
    ([2, 0, 2, 0], [12, 10, 11, 13], [(12, 11), (10, 13)]),
])
def test_plan_reorder(parents, new, copies):
    got, moved = beam.plan_reorder([10, 11, 12, 13], parents)
    assert got.tolist() == new and moved == copies


def test_plan_reorder_of_random_parents_keeps_every_beam():
    rng = np.random.default_rng(5)
    for _ in range(200):
        k = int(rng.integers(1, 20))
        slots = rng.permutation(64)[:k].tolist()
        parents = rng.integers(0, k, k).tolist()
        new, copies = beam.plan_reorder(slots, parents)
        assert sorted(new.tolist()) == sorted(slots)
        content = {s: i for i, s in enumerate(slots)}
        for src, dst in copies:  # a source is never overwritten, so the order is free
            assert src not in {d for _, d in copies}
            content[dst] = content[src]
        assert [content[s] for s in new.tolist()] == parents


@pytest.mark.parametrize("head_dim,unit", [(64, 8), (128, 8), (256, 4)])
def test_prefix_split_plan_covers_every_page(head_dim, unit):
    rng = np.random.default_rng(head_dim)
    for _ in range(300):
        tiles = rng.integers(1, 2000, int(rng.integers(1, 9))).tolist()
        heads, sms = int(rng.integers(1, 9)), int(rng.integers(1, 149))
        pps, splits = paged.prefix_split_plan(tiles, heads, head_dim, sms)
        assert pps % unit == 0 and pps * splits >= max(tiles) > pps * (splits - 1)
        ctas = sum(-(-t // pps) for t in tiles) * heads
        assert ctas <= max(sms, len(tiles) * heads)
    assert paged.prefix_split_plan([], 2, head_dim, 148)[1] == 1
    assert paged.prefix_split_plan([100], 2, head_dim, 148, unit + 1) == \
        (2 * unit, -(-100 // (2 * unit)))


def test_tail_split_plan_covers_every_page():
    for batch in (1, 7, 64):
        for pages in (1, 5, 64, 4096):
            for total in (None, batch, batch * pages):
                pps, splits = paged.tail_split_plan(batch, 16, 2, pages, None, total, 148)
                assert 4 <= pps <= 16 and pps * splits >= pages > pps * (splits - 1)
    assert paged.tail_split_plan(4, 16, 2, 40, 7, None, 148) == (7, 6)


def test_prefix_groups_tables():
    groups = paged.PrefixGroups([([0, 2, 3], 49), ([1], 64), ([5, 4], 8)], 7, 16, 2, 128,
                                device="cpu", sms=148)
    assert groups.ntiles == 1 and groups.tiles.tolist() == [0, 3, 3, 0]
    assert groups.members.tolist() == [0, 2, 3]
    assert groups.first_page.tolist() == [3, 0, 3, 3, 0, 0, 0]
    big = paged.PrefixGroups([(range(40), 160)], 40, 16, 2, 128, device="cpu", sms=148)
    tiles = big.tiles.view(-1, 4).tolist()  # 128 / 8 = 16 members a tile, spread evenly
    assert [t[1] for t in tiles] == [13, 13, 14] and [t[0] for t in tiles] == [0, 13, 26]
    few, many = big.splits(1000), big.splits(0)
    assert few[0] >= many[0] and big.splits(None) == few
    for bad in ([([0, 7], 16)], [([0, 0], 16)], [([0, 1], 16), ([1, 2], 16)], [([0, 1], -1)]):
        with pytest.raises(ValueError):
            paged.PrefixGroups(bad, 7, 16, 2, 128, device="cpu", sms=148)
    with pytest.raises(ValueError):
        paged.PrefixGroups([], 7, 10, 4, 128, device="cpu", sms=148)
    with pytest.raises(ValueError):
        paged.PrefixGroups([], 7, 16, 2, 96, device="cpu", sms=148)


def test_replace_and_common_prefixes():
    blocks = BlockManager(num_pages=32, max_seqs=6, page_size=16, max_pages_per_seq=8)
    a, b, c = (blocks.admit(name, 40) for name in "abc")
    assert blocks.common_prefixes() == []
    shared = blocks.pages[a][:2]
    before, count = blocks.free_pages, blocks.sharing
    blocks.share(shared)
    own = blocks.take_pages(1)
    blocks.replace(b, shared + own, 40)
    assert blocks.free_pages == before - 1 + 3 and blocks.sharing == count + 1
    assert blocks.common_prefixes() == [([a, b], 2)]
    assert blocks.table[b, :3].tolist() == shared + own and not blocks.table[b, 3:].any()
    with pytest.raises(ValueError):
        blocks.replace(b, shared, 40)
    with pytest.raises(ValueError):
        blocks.replace(c, shared * 5, 160)
    assert blocks.pages[b] == shared + own
    for slot in (a, b, c):
        blocks.release(slot)
    assert blocks.free_pages == 32 and not blocks.refcount.any()


def test_group_operators_are_registered_with_their_mutations():
    expect = {"rotary_append": ["kv_pool"], "shared_prefix_attention": [], "beam_select": [],
              "reorder_rows": ["pools"]}
    assert set(torch_ops.GROUP_OPERATORS) == set(expect)
    for name, mutated in expect.items():
        op = getattr(torch.ops.shellcache, name).default
        assert [a.name for a in op._schema.arguments
                if a.alias_info and a.alias_info.is_write] == mutated


def test_group_fake_kernels_propagate_shapes():
    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    ops = torch.ops.shellcache
    with FakeTensorMode():
        make = lambda *shape, dtype=bf: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
        q, k, pool = make(5, 16, 128), make(5, 2, 128), make(64, 2, 2, 16, 128)
        out = ops.rotary_append(q, k, k, make(1, 5, dtype=i32), pool,
                                make(5, dtype=torch.int64), 64)
        assert out.shape == q.shape and out.dtype == bf
        out = ops.shared_prefix_attention(q, pool, make(5, 8, dtype=i32), make(5, dtype=i32), 0.1,
                                          [0, 1], [2], [32])
        assert out.shape == q.shape
        best, parents, tokens = ops.beam_select(make(3, 4, 1000), make(3, 4, dtype=f32), 6)
        assert best.shape == parents.shape == tokens.shape == (3, 6)
        assert (best.dtype, parents.dtype, tokens.dtype) == (f32, i32, i32)
        slots = make(3, 4, dtype=i32)
        assert ops.reorder_rows([make(2, 12, 64)], slots, slots).shape == slots.shape


def test_freed_by_counts_pages_that_nobody_else_owns():
    blocks = BlockManager(num_pages=32, max_seqs=6, page_size=16, max_pages_per_seq=8)
    a, b = blocks.admit("a", 40), blocks.admit("b", 20)
    shared = blocks.pages[a][:2]
    blocks.share(shared)
    c = blocks.adopt("c", shared + blocks.take_pages(1), 40)
    for slots, pages in (([a], 1), ([b], 2), ([c], 1), ([a, c], 4), ([a, b, c], 6), ([], 0)):
        assert blocks.freed_by(slots) == pages


@pytest.mark.parametrize("kv_heads", [1, 2, 8])
@pytest.mark.parametrize("prefix_splits", [1, 37, 148])
def test_tail_split_plan_keeps_to_the_parts_that_the_entry_takes(kv_heads, prefix_splits):
    """Own pages of 64k to 5M tokens, with and without their number known."""
    most = paged.MOST_PARTS - prefix_splits
    for pages in (4000, 4079, 4080, 4200, 4735, 8200, 9471, 16300, 18750, 65536, 327680):
        for batch, total in ((1, pages), (2, pages + 3), (64, pages + 640), (8, None)):
            pps, splits = paged.tail_split_plan(batch, 16, kv_heads, pages, None, total, 148, most)
            assert splits <= most and pps * splits >= pages > pps * (splits - 1)
            free = paged.tail_split_plan(batch, 16, kv_heads, pages, None, total, 148)
            assert free == (pps, splits) or free[1] > most


@pytest.mark.parametrize("batch", [2, 64, 256, 1024, 5000])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (16, 1, 256), (32, 8, 128), (8, 8, 64)])
def test_parts_of_one_long_sequence_in_a_large_batch_stay_small(batch, heads, kv_heads, dim):
    """Two rows on a long prefix, one row of 128k own tokens, the others short."""
    groups = paged.PrefixGroups([([0, 1], 200_000)], batch, heads, kv_heads, dim, device="cpu",
                                sms=148)
    part = 4 * batch * heads * dim
    most = max(paged.PART_BYTES, 8 * part)
    for own in (None, batch + 8192):
        pps, splits = groups.splits(own)
        assert splits * part <= most and pps * splits >= 12500 > pps * (splits - 1)
        pps, splits = paged.tail_split_plan(batch, heads, kv_heads, 8192, None, own, 148,
                                            groups.most_splits)
        assert splits * part <= most and pps * splits >= 8192 > pps * (splits - 1)


@pytest.mark.parametrize("beams,vocab", [(1, 2 ** 31 - 1), (1, 2 ** 31 - 2 ** 14 + 1), (2, 2 ** 30),
                                         (64, 2 ** 25 + 1)])
def test_beam_select_refuses_more_than_its_indices_hold(beams, vocab):
    """Refused by the entry point before it looks at the memory or the GPU."""
    unsupported = 2
    host = ctypes.create_string_buffer(512)
    at = (ctypes.addressof(host) + 255) // 256 * 256
    code = _capi.lib().sc_beam_select(at, 0, vocab, at, None, 0, at, at, at, at, 2 ** 60, 1, beams,
                                      vocab, 4, None)
    assert code == unsupported and "beams * vocab" in _capi.last_error()
