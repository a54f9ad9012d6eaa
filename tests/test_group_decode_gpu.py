"""Beam search over the paged engine (group_decode.BeamSearch, HybridCacheEngine.reorder).

Bars. A beam's tokens forced through a single sequence of a fresh engine give its score:
the two differ in batch shapes only (bf16 GEMM and attention rounding; the resident tests
measured up to 0.005 a step for such a change, bar 0.02 a step). Pages and slots are exact:
shared pages counted once per owner, everything back at the end. Reordered rows and pages
are bit copies.
"""

import numpy as np
import pytest
import torch

from shellsmith_b200 import paged, rotary
from shellsmith_b200.engine import HybridCacheEngine, HybridConfig
from shellsmith_b200.group_decode import BeamSearch
from shellsmith_b200.resident import ToyHybridModel

pytestmark = pytest.mark.gpu
TOL = 0.02


def _cfg(**kw):
    base = dict(layers=4, gdn_key_heads=2, gdn_value_heads=4, q_heads=8, kv_heads=2, head_dim=128,
                max_seqs=10, num_pages=200, max_context=512, snapshot_rows=2, gdn_taps=True)
    return HybridConfig(**{**base, **kw})


def _search(cuda, cfg, model, stop=None):
    eng = HybridCacheEngine(cfg, device=cuda)
    plan = rotary.RotaryPlan(cfg.head_dim, cfg.head_dim // 2, sections=(12, 10, 10)
                             if cfg.head_dim == 128 else None, device=cuda)
    w = (1 + 0.1 * torch.randn(cfg.head_dim, generator=torch.Generator().manual_seed(1)))
    w = w.to(cuda, torch.bfloat16)
    return eng, BeamSearch(eng, model, plan, q_weight=w, k_weight=w, stop_token=stop)


def _forced_score(cuda, cfg, model, prompt, tokens):
    """log-probability of `tokens` after `prompt`, one sequence by itself."""
    eng, one = _search(cuda, cfg, model)
    one.start(prompt, 1)
    total = 0.0
    for i, t in enumerate(tokens):
        total += float(torch.log_softmax(one._logits.double(), -1)[0, t])
        one.beams[0].tokens = list(tokens[:i + 1])
        if i + 1 < len(tokens):
            one.step()
    return total


@pytest.mark.parametrize("beams,prompt_len,steps", [(4, 37, 20), (3, 64, 7), (8, 5, 6), (1, 20, 5)])
def test_beam_scores_are_their_tokens_log_probabilities(cuda, beams, prompt_len, steps):
    cfg = _cfg()
    model = ToyHybridModel(cfg, device=cuda)
    rng = np.random.default_rng(prompt_len)
    prompt = [int(t) for t in rng.integers(0, model.vocab, prompt_len)]
    eng, search = _search(cuda, cfg, model)
    free = eng.blocks.free_pages
    found = search.search(prompt, beams, steps)
    assert len(found) == beams and len({tuple(b.tokens) for b in found}) == beams
    assert [b.score for b in found] == sorted((b.score for b in found), reverse=True)
    full = prompt_len // cfg.page_size
    if beams > 1 and full:  # the prompt's full pages are shared by every beam
        first = [eng.blocks.pages[s][:full] for s in search.slots]
        assert all(p == first[0] for p in first)
        assert (eng.blocks.refcount[first[0]] == beams).all()
        assert eng.prefix_groups().ntiles >= 1
    for b in found:
        assert len(b.tokens) == steps
        want = _forced_score(cuda, cfg, model, prompt, b.tokens)
        assert abs(b.score - want) <= TOL * steps, (b.score, want)
    search.close()
    assert eng.blocks.free_pages == free and not eng.blocks.refcount.any()


def test_one_beam_is_greedy(cuda):
    cfg = _cfg()
    model = ToyHybridModel(cfg, device=cuda)
    eng, search = _search(cuda, cfg, model)
    search.start([3, 1, 4, 1, 5], 1)
    for _ in range(5):
        search.step()
    tokens = search.beams[0].tokens
    assert len(tokens) == 6
    eng2, again = _search(cuda, cfg, model)
    again.start([3, 1, 4, 1, 5], 1)
    for i in range(6):
        assert again.beams[0].tokens[:i + 1] == tokens[:i + 1]
        again.step()


def test_stop_token_finishes_a_beam(cuda):
    """The most likely first token as stop token: that beam keeps its score and tokens."""
    cfg = _cfg()
    model = ToyHybridModel(cfg, device=cuda)
    eng, probe = _search(cuda, cfg, model)
    probe.start([7, 8, 9], 1)
    stop = probe.beams[0].tokens[0]
    eng, search = _search(cuda, cfg, model, stop=stop)
    search.start([7, 8, 9], 3)
    done = [b for b in search.beams if b.finished]
    assert len(done) == 1 and done[0].tokens == [stop]
    score = done[0].score
    for _ in range(4):
        search.step()
    still = [b for b in search.beams if b.tokens == [stop]]
    assert len(still) <= 1 and all(b.score == score for b in still)
    for b in search.beams:
        assert stop not in b.tokens[:-1]


def test_reorder_moves_state_taps_and_pages(cuda):
    cfg = _cfg()
    eng = HybridCacheEngine(cfg, device=cuda)
    slots = [eng.admit(i, 20 + 5 * i) for i in range(4)]
    eng.state.copy_(torch.randn_like(eng.state))
    eng.taps.copy_(torch.randn(eng.taps.shape, device=cuda).to(torch.bfloat16))
    eng.kv.copy_(torch.randn(eng.kv.shape, device=cuda).to(torch.bfloat16))
    state, taps = eng.state.clone(), eng.taps.clone()
    read = lambda s, n: [paged.kv_gather(eng.kv[i], torch.from_numpy(  # noqa: E731
        eng.blocks.prompt_slots(s, 0, n)).to(cuda)) for i in range(eng.kv.shape[0])]
    before = [read(s, 20 + 5 * i) for i, s in enumerate(slots)]
    parents = [2, 2, 0, 2]
    new = eng.reorder(slots, parents)
    assert new == [slots[2], slots[1], slots[0], slots[3]]
    for j, p in enumerate(parents):
        assert torch.equal(eng.state[:, new[j]], state[:, slots[p]])
        assert torch.equal(eng.taps[:, new[j]], taps[:, slots[p]])
        n = 20 + 5 * p
        assert int(eng.blocks.lengths[new[j]]) == n
        for (k, v), (k0, v0) in zip(read(new[j], n), before[p]):
            assert torch.equal(k, k0) and torch.equal(v, v0)
    shared = eng.blocks.pages[slots[2]][0]
    assert eng.blocks.refcount[shared] == 3 and eng.blocks.refcount[eng.blocks.pages[slots[2]][1]] == 1
    assert eng.blocks.common_prefixes() == [([slots[1], slots[2], slots[3]], 1)]
    for s in new:
        eng.release(s)
    assert not eng.blocks.refcount.any()
    with pytest.raises(ValueError):
        eng.reorder(slots, parents)
    with pytest.raises(ValueError):
        eng.reorder([0], [1])


def test_reorder_without_free_pages_changes_nothing(cuda):
    cfg = _cfg(num_pages=4)
    eng = HybridCacheEngine(cfg, device=cuda)
    slots = [eng.admit(i, 20) for i in range(2)]
    pages = [list(eng.blocks.pages[s]) for s in slots]
    with pytest.raises(MemoryError):
        eng.reorder(slots, [0, 0])
    assert [eng.blocks.pages[s] for s in slots] == pages
    assert eng.reorder(slots, [1, 0]) == [slots[1], slots[0]]  # a permutation needs none


def test_errors_leave_no_pages_behind(cuda):
    cfg = _cfg(max_seqs=3)
    model = ToyHybridModel(cfg, device=cuda)
    eng, search = _search(cuda, cfg, model)
    with pytest.raises(ValueError):
        search.start([], 2)
    with pytest.raises(ValueError):
        search.start([1], 65)
    with pytest.raises(MemoryError):
        search.start([1] * 40, 4)  # three slots
    search.close()
    assert not eng.blocks.refcount.any() and not eng.blocks.active.any()
    search.start([1] * 40, 3)
    with pytest.raises(ValueError):
        search.start([1], 1)
    with pytest.raises(ValueError):
        BeamSearch(HybridCacheEngine(_cfg(gdn_taps=False), device=cuda), model, search.plan)


@pytest.mark.parametrize("axes,staged", [(1, None), (3, None), (1, [0, 2, 5]), (3, [5, 3])])
def test_group_attention_equals_the_plain_layer(cuda, axes, staged):
    """A staged batch (or a part of it) of forks, a stranger and an empty row: the same
    result as the layer that reads every sequence's pages for itself."""
    cfg = _cfg(layers=4, head_dim=256, q_heads=16)
    eng = HybridCacheEngine(cfg, device=cuda)
    a = eng.admit("a", 100)
    layer = cfg.attention_layers[0]
    kv = torch.randn((2, 100, 2, 256), device=cuda).to(torch.bfloat16)
    eng.write_prompt_kv(a, layer, kv[0], kv[1])
    snap = eng.snapshot(a)
    forks = [eng.fork(snap) for _ in range(3)]
    gone = eng.admit("gone", 30)
    other = eng.admit("other", 30)
    eng.write_prompt_kv(other, layer, kv[1][:30].contiguous(), kv[0][:30].contiguous())
    eng.release(gone)
    eng.begin_step(staged)
    n = eng.rows
    q = torch.randn((n, 16, 256), device=cuda).to(torch.bfloat16)
    k, v = torch.randn((2, n, 2, 256), device=cuda).to(torch.bfloat16)
    plan = rotary.RotaryPlan(256, 64, sections=(12, 10, 10) if axes == 3 else None, device=cuda)
    turned = eng.append_rotary(layer, q, k, v, plan)
    out = torch.empty_like(q)
    eng.group_attention_layer(layer, turned, out)
    assert eng.prefix_groups().ntiles == 1
    want = paged.paged_decode_attention(turned, eng.kv[eng.attn_index[layer]], eng.table[:n],
                                        eng.ctx_len[:n], eng.scale)
    # Both round P to bf16 in other places: 2^-8 of sum p |v| (below 2) each, and the output.
    assert (out.float() - want.float()).abs().max() <= 3 * 2.0 ** -8 * 2
    assert not out[gone].any() and (staged is None or not out[1].any())
