"""Beam search and reordering on a pool that holds just what they need.

Pages are exact. A search that had to wait for a page goes on as one that never did: the
same launches on the same values, so the same bits.
"""

import pytest
import torch
from test_group_decode_gpu import _cfg, _search

from shellsmith_b200 import _capi, paged
from shellsmith_b200.block_manager import OutOfPages
from shellsmith_b200.engine import HybridCacheEngine
from shellsmith_b200.resident import ToyHybridModel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length,beams", [(37, 4), (37, 2), (33, 8), (48, 3), (5, 5)])
def test_a_search_fits_the_pages_that_start_asks_for(cuda, length, beams):
    need = -(-length // 16) + (beams if length % 16 else 0)
    prompt = [3 + i % 90 for i in range(length)]
    cfg = _cfg(num_pages=need)
    model = ToyHybridModel(cfg, device=cuda)
    eng, search = _search(cuda, cfg, model)
    search.start(prompt, beams)
    for _ in range(-length % 16):  # up to the page's end: no further page is needed
        search.step()
    assert all(len(b.tokens) == 1 + -length % 16 for b in search.beams)
    before = (list(search.slots), search._scores.clone(), [list(b.tokens) for b in search.beams],
              eng.blocks.lengths.copy(), eng.blocks.free_pages)
    if eng.blocks.free_pages < beams:
        with pytest.raises(OutOfPages):
            search.step()
        assert before[0] == search.slots and torch.equal(before[1], search._scores)
        assert before[2] == [b.tokens for b in search.beams]
        assert (before[3] == eng.blocks.lengths).all() and before[4] == eng.blocks.free_pages
    search.close()
    assert eng.blocks.free_pages == need and not eng.blocks.refcount.any()
    small = _cfg(num_pages=need - 1)
    eng, search = _search(cuda, small, model)
    with pytest.raises(MemoryError):
        search.start(prompt, beams)
    assert not search.slots and eng.blocks.free_pages == need - 1


def test_a_search_goes_on_when_there_is_room_again(cuda):
    prompt, beams = [3 + i % 90 for i in range(37)], 4
    found = []
    for fills in (True, False):
        cfg = _cfg(num_pages=30)
        model = ToyHybridModel(cfg, device=cuda)
        eng, search = _search(cuda, cfg, model)
        search.start(prompt, beams)
        for _ in range(20):
            if int(eng.blocks.lengths[search.slots[0]]) == 48:  # the next token takes a page
                other = eng.admit("other", 16 * eng.blocks.free_pages if fills else 16)
                if fills:
                    with pytest.raises(OutOfPages):
                        search.step()
                eng.release(other)
            search.step()
        assert [len(b.tokens) for b in search.beams] == [21] * beams
        found.append(([b.tokens for b in search.beams], search._scores.clone()))
    assert found[0][0] == found[1][0] and torch.equal(found[0][1], found[1][1])


def test_start_without_a_snapshot_row_opens_nothing(cuda):
    cfg = _cfg(snapshot_rows=1)
    model = ToyHybridModel(cfg, device=cuda)
    eng, search = _search(cuda, cfg, model)
    other = eng.admit("other", 10)
    snap = eng.snapshot(other)
    free = eng.blocks.free_pages
    with pytest.raises(MemoryError):
        search.start([1, 2, 3], 2)
    assert not search.slots and eng.blocks.free_pages == free
    search.start([1, 2, 3], 1)            # one beam needs none
    search.close()
    eng.drop_snapshot(snap)
    search.start([1, 2, 3], 2)
    search.close()
    assert eng.blocks.free_pages == free + 1


def test_an_error_in_start_opens_nothing(cuda, monkeypatch):
    cfg = _cfg()
    model = ToyHybridModel(cfg, device=cuda)
    eng, search = _search(cuda, cfg, model)
    monkeypatch.setattr(eng, "reorder", lambda *a, **kw: 1 / 0)
    free, rows = eng.blocks.free_pages, eng.free_snapshot_rows
    with pytest.raises(ZeroDivisionError):
        search.start([1, 2, 3], 3)
    assert not search.slots and not search.beams
    assert eng.blocks.free_pages == free and eng.free_snapshot_rows == rows


def test_reorder_takes_the_pages_that_its_beams_give_back(cuda):
    eng = HybridCacheEngine(_cfg(num_pages=8), device=cuda)
    slots = [eng.admit(i, 20) for i in range(4)]
    eng.kv.copy_(torch.randn(eng.kv.shape, device=cuda).to(torch.bfloat16))
    kv = eng.kv.clone()
    pages = [list(eng.blocks.pages[s]) for s in slots]
    with pytest.raises(MemoryError):
        eng.reorder(slots, [1, 1, 3, 3])
    assert [eng.blocks.pages[s] for s in slots] == pages
    new = eng.reorder(slots, [1, 1, 3, 3], reuse_pages=True)
    assert new == [slots[1], slots[0], slots[3], slots[2]]
    for j, p in enumerate([1, 1, 3, 3]):
        mine = eng.blocks.pages[new[j]]
        assert mine[0] == pages[p][0] and eng.blocks.refcount[mine].tolist() == [2, 1]
        for i in range(2):
            assert torch.equal(eng.kv[:, mine[i]], kv[:, pages[p][i]])
    assert eng.blocks.free_pages == 2     # two full pages went, the partial ones came back


@pytest.mark.parametrize("laid_out", [False, True])
@pytest.mark.parametrize("low_slot", [False, True])
def test_sequences_that_come_between_staging_and_attention(cuda, laid_out, low_slot):
    """A fork after begin_step, into a slot past the staged rows or below them: the staged rows
    attend to what was staged (a lower slot would lead the group with a table row that the
    device does not have)."""
    cfg = _cfg()
    eng = HybridCacheEngine(cfg, device=cuda)
    first = eng.admit("first", 40)        # holds slot 0
    a = eng.admit("a", 100)
    eng.kv.copy_(torch.randn(eng.kv.shape, device=cuda).to(torch.bfloat16))
    snap = eng.snapshot(a)
    for _ in range(2):
        eng.fork(snap)
    if low_slot:
        eng.release(first)
    eng.begin_step()
    if laid_out:
        assert eng.prefix_groups().ntiles == 1
    new = eng.fork(snap)
    assert new == (0 if low_slot else eng.rows)
    n, layer = eng.rows, cfg.attention_layers[0]
    q = torch.randn((n, cfg.q_heads, cfg.head_dim), device=cuda).to(torch.bfloat16)
    out = torch.empty_like(q)
    eng.group_attention_layer(layer, q, out)
    want = paged.paged_decode_attention(q, eng.kv[eng.attn_index[layer]], eng.table[:n],
                                        eng.ctx_len[:n], eng.scale)
    _capi.check_device()
    # Both round P to bf16 in other places: 2^-8 of sum p |v| (below 2) each, and the output.
    assert (out.float() - want.float()).abs().max() <= 3 * 2.0 ** -8 * 2
    eng.begin_step()
    assert eng.prefix_groups().ntiles == 1 and len(eng.prefix_groups().members) == 4


def test_search_refuses_less_than_a_token(cuda):
    cfg = _cfg()
    eng, search = _search(cuda, cfg, ToyHybridModel(cfg, device=cuda))
    for count in (0, -3):
        with pytest.raises(ValueError):
            search.search([1, 2, 3], 2, count)
    assert not search.slots
    assert all(len(b.tokens) == 1 for b in search.search([1, 2, 3], 2, 1))
