"""Beam selection and row reordering (beam.py) on the GPU.

Selection bars, against scores in 64 bits. An fp32 score is score + ((x - m) - L): x - m
and the two sums round once each (2^-24 of their size) and L = log of an fp32 sum of at
most 2^18 terms, summed over 64 a thread and then in a tree, each term an exponential to 2
units (2^-22) of an argument rounded twice: relative error of the sum below 2^-19. With
sizes up to 2^6 here: |error| <= 3 * 2^-24 * 2^6 + 2^-19 < 1.4e-5; TOL = 2e-5. The places
are checked by their 64-bit scores and, where scores tie exactly, by equality: lowest
index first. Reordering moves bits and is exact.
"""

import numpy as np
import pytest
import torch

from shellsmith_b200 import _capi, beam

pytestmark = pytest.mark.gpu

TOL = 2e-5


def _scores64(logits, scores, finished=None, pad=0):
    x = logits.double().cpu().numpy()
    G, K, V = x.shape
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        s = scores.double().cpu().numpy()[..., None] + (
            x - m - np.log(np.exp(x - m).sum(-1, keepdims=True)))
    s[np.isnan(s)] = -np.inf
    if finished is not None:
        for g, k in np.argwhere(finished.cpu().numpy()):
            s[g, k] = -np.inf
            s[g, k, pad] = float(scores[g, k])
    return s.reshape(G, K * V)


def _check(logits, scores, n, finished=None, pad=0):
    got, parents, tokens = beam.beam_select(logits, scores, n, finished=finished, pad_token=pad)
    G, K, V = logits.shape
    assert got.shape == parents.shape == tokens.shape == (G, n)
    assert parents.dtype == tokens.dtype == torch.int32 and got.dtype == torch.float32
    want = _scores64(logits, scores, finished, pad)
    out = got.double().cpu().numpy()
    at = parents.cpu().numpy().astype(np.int64) * V + tokens.cpu().numpy()
    assert (0 <= tokens.cpu().numpy()).all() and (tokens.cpu().numpy() < V).all()
    best = -np.sort(-want, axis=1, kind="stable")[:, :n]
    order = np.argsort(-want, axis=1, kind="stable")[:, :n]
    for g in range(G):
        assert len(set(at[g])) == n
        assert (out[g][:-1] >= out[g][1:]).all()
        fin = np.isfinite(best[g])
        np.testing.assert_allclose(out[g][fin], best[g][fin], rtol=0, atol=TOL)
        np.testing.assert_allclose(want[g, at[g]][fin], out[g][fin], rtol=0, atol=TOL)
        assert np.array_equal(out[g][~fin], best[g][~fin])          # -inf (or +inf) exactly
        assert np.array_equal(at[g][~fin], order[g][~fin])          # then lowest index first
        ties = out[g][:-1] == out[g][1:]
        assert (at[g][:-1][ties] < at[g][1:][ties]).all()
    _capi.check_device()
    return got, parents, tokens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,K,V,n", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 6), (1, 4, 4096, 8),
                                     (3, 5, 5001, 10), (2, 2, 70003, 64), (1, 64, 1000, 64),
                                     (4, 1, 33000, 16), (9, 8, 40001, 16)])
def test_select_matches_64_bits(cuda, dtype, G, K, V, n):
    logits = (torch.randn((G, K, V), device=cuda) * 2.5).to(dtype)
    scores = -torch.rand((G, K), device=cuda) * 30
    _check(logits, scores, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_select_strided_and_unaligned_rows(cuda, dtype):
    base = (torch.randn((3, 4, 9001 + 13), device=cuda) * 3).to(dtype)
    scores = -torch.rand((3, 4), device=cuda) * 10
    for first in (0, 1, 5):
        view = base[..., first:first + 9001]
        got = _check(view, scores, 8)
        want = beam.beam_select(view.contiguous(), scores, 8)
        # Another alignment cuts the row into other chunks: the sums round differently.
        assert (got[0] - want[0]).abs().max() <= 2 * TOL
    _check(base[..., 3:8000], scores, 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [50, 5000, 40000])
def test_equal_logits_give_the_lowest_places(cuda, dtype, V):
    logits = torch.full((2, 3, V), 1.5, device=cuda, dtype=dtype)
    scores = torch.zeros((2, 3), device=cuda)
    n = 40
    got, parents, tokens = beam.beam_select(logits, scores, n)
    assert (parents == 0).all()
    assert torch.equal(tokens.cpu(), torch.arange(n, dtype=torch.int32).expand(2, n))
    logits[0, 2, V // 2] = 3.0          # one better token, then the ties
    got, parents, tokens = beam.beam_select(logits, scores, n)
    assert parents[0, 0] == 2 and tokens[0, 0] == V // 2
    # Beam 2's other scores fell with its larger sum; beams 0 and 1 tie.
    assert (parents[0, 1:] == 0).all() and torch.equal(tokens[0, 1:].cpu(),
                                                       torch.arange(n - 1, dtype=torch.int32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_logits(cuda, dtype):
    """Rows masked by -inf and by the type's lowest value, rows that leave nothing."""
    V, K = 20011, 6
    logits = (torch.randn((2, K, V), device=cuda) * 2).to(dtype)
    scores = -torch.arange(K, device=cuda, dtype=torch.float32).expand(2, K).contiguous()
    keep = torch.zeros(V, dtype=torch.bool, device=cuda)
    keep[[3, 9000, 9001, 20010]] = True
    logits[:, 0] = torch.where(keep, logits[:, 0], -float("inf"))
    logits[:, 1] = torch.where(keep, logits[:, 1], torch.finfo(dtype).min)
    logits[:, 2] = -float("inf")
    logits[0, 3, 17] = float("nan")
    logits[1, 3, 17] = float("inf")
    _check(logits, scores, 12)
    only = logits[:, :1].contiguous()
    got, parents, tokens = _check(only, scores[:, :1].contiguous(), 9)
    assert torch.isinf(got[:, 4:]).all() and tokens[0, 4:].tolist() == [0, 1, 2, 4, 5]
    got, _, tokens = _check(logits[:, 2:3].contiguous(), scores[:, :1].contiguous(), 5)
    assert torch.isneginf(got).all() and tokens[0].tolist() == [0, 1, 2, 3, 4]
    _check(logits[:, 3:4].contiguous(), scores[:, :1].contiguous(), 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_finished_and_dead_beams(cuda, dtype):
    G, K, V = 3, 5, 6007
    logits = (torch.randn((G, K, V), device=cuda) * 2).to(dtype)
    scores = -torch.rand((G, K), device=cuda) * 8
    finished = torch.zeros((G, K), dtype=torch.bool, device=cuda)
    finished[0, 1] = finished[0, 4] = finished[1] = True
    scores[2, 1:] = -float("inf")      # the first step: one live beam
    scores[0, 2] = float("nan")
    _check(logits, scores, 10, finished, pad=2)
    got, parents, tokens = beam.beam_select(logits[1:2], scores[1:2].contiguous(), 7,
                                            finished=finished[1:2].contiguous(), pad_token=2)
    order = torch.argsort(scores[1], descending=True)
    assert torch.equal(parents[0, :5].long(), order) and (tokens[0, :5] == 2).all()
    assert torch.equal(got[0, :5], scores[1][order])
    assert parents[0, 5:].tolist() == [0, 0] and tokens[0, 5:].tolist() == [0, 1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_that_round_together_keep_index_order(cuda, dtype):
    """At -1e9 an fp32 step is 64: every token of such a beam has the same score, and the
    lowest indices win although their logits are not the largest."""
    V = 30011
    logits = (torch.randn((2, 3, V), device=cuda) * 2).to(dtype)
    scores = torch.full((2, 3), -1e9, device=cuda)
    got, parents, tokens = beam.beam_select(logits, scores, 20)
    assert (got == -1e9).all() and (parents == 0).all()
    assert torch.equal(tokens.cpu(), torch.arange(20, dtype=torch.int32).expand(2, 20))
    scores[:, 1] = -3.0                # one live beam among them, fewer tokens than asked
    logits[:, 1] = torch.where(torch.arange(V, device=cuda) < 4, logits[:, 1], -float("inf"))
    finished = torch.zeros((2, 3), dtype=torch.bool, device=cuda)
    finished[1, 0] = True
    got, parents, tokens = beam.beam_select(logits, scores, 10, finished=finished, pad_token=7)
    assert (parents[:, :4] == 1).all() and (got[:, 4:] == -1e9).all()
    assert parents[0, 4:].tolist() == [0] * 6 and tokens[0, 4:].tolist() == list(range(6))
    assert parents[1, 4:].tolist() == [0] + [2] * 5 and tokens[1, 4:].tolist() == [7, 0, 1, 2, 3, 4]


def test_clustered_logits(cuda):
    """Runs of large neighbours: many survivors in few threads, cut to the segment."""
    for dtype in (torch.bfloat16, torch.float32):
        for V in (4096, 60000):
            x = torch.linspace(-20, 10, V, device=cuda).to(dtype).expand(2, 2, V).contiguous()
            scores = torch.tensor([[0.0, -0.5], [-1.0, -40.0]], device=cuda)
            _check(x, scores, 64)
            _check(x.flip(-1).contiguous(), scores, 64)


def test_select_refusals(cuda):
    x = torch.zeros((2, 3, 50), device=cuda)
    s = torch.zeros((2, 3), device=cuda)
    with pytest.raises(TypeError):
        beam.beam_select(x.half(), s, 4)
    with pytest.raises(ValueError):
        beam.beam_select(x[0], s, 4)
    with pytest.raises(ValueError):
        beam.beam_select(x, s[:1], 4)
    with pytest.raises(ValueError):
        beam.beam_select(x.transpose(1, 2), torch.zeros((2, 50), device=cuda), 4)
    with pytest.raises(ValueError):
        beam.beam_select(x.cpu(), s, 4)
    with pytest.raises(TypeError):
        beam.beam_select(x, s, 4, finished=torch.zeros((2, 3), device=cuda))
    for n in (0, 65, 151):
        with pytest.raises(_capi.ShellcacheError):
            beam.beam_select(x, s, n)
    with pytest.raises(_capi.ShellcacheError):
        beam.beam_select(x, s, 4, finished=torch.zeros((2, 3), dtype=torch.bool, device=cuda),
                         pad_token=50)
    with pytest.raises(_capi.ShellcacheError):
        beam.beam_select(torch.zeros((1, 65, 9), device=cuda), torch.zeros((1, 65), device=cuda), 4)
    assert beam.beam_select(x[:0], s[:0], 4)[0].shape == (0, 4)


# ---------------------------------------------------------------- reordering
@pytest.mark.parametrize("G,K", [(1, 1), (1, 2), (3, 4), (5, 8), (2, 33), (1, 64)])
def test_reorder_follows_the_beams(cuda, G, K):
    rng = np.random.default_rng(G * 100 + K)
    rows = G * K + 3
    state = torch.randn((3, rows, 2, 8, 24), device=cuda)
    taps = torch.randn((2, rows, 4, 1001 * 8), device=cuda).to(torch.bfloat16)
    s0, t0 = state.clone(), taps.clone()
    slots = rng.permutation(rows)[:G * K].reshape(G, K).astype(np.int32)
    parents = rng.integers(0, K, (G, K)).astype(np.int32)
    new = beam.reorder_rows([state, taps], torch.from_numpy(slots).to(cuda),
                            torch.from_numpy(parents).to(cuda)).cpu().numpy()
    changed = set()
    for g in range(G):
        want, copies = beam.plan_reorder(slots[g], parents[g])
        assert np.array_equal(new[g], want)
        assert len(copies) == K - len(set(parents[g].tolist()))
        changed |= {d for _, d in copies}
        for j in range(K):
            src = int(slots[g, parents[g, j]])
            assert torch.equal(state[:, int(new[g, j])], s0[:, src])
            assert torch.equal(taps[:, int(new[g, j])], t0[:, src])
    for r in set(range(rows)) - changed:
        assert torch.equal(state[:, r], s0[:, r]) and torch.equal(taps[:, r], t0[:, r])
    _capi.check_device()


def test_reorder_extremes(cuda):
    state = torch.arange(2 * 6 * 8, dtype=torch.float32, device=cuda).view(2, 6, 8)
    keep = state.clone()
    slots = torch.tensor([[4, 1, 0, 5]], dtype=torch.int32, device=cuda)
    same = torch.tensor([[3, 1, 0, 2]], dtype=torch.int32, device=cuda)   # a permutation: no copy
    new = beam.reorder_rows([state], slots, same)
    assert torch.equal(state, keep) and new.tolist() == [[5, 1, 4, 0]]
    one = torch.tensor([[2, 2, 2, 2]], dtype=torch.int32, device=cuda)    # one survivor
    new = beam.reorder_rows([state], slots, one)
    assert new.tolist() == [[0, 4, 1, 5]]
    assert all(torch.equal(state[:, r], keep[:, 0]) for r in (0, 4, 1, 5))
    assert torch.equal(state[:, 2:4], keep[:, 2:4])
    assert beam.reorder_rows([], slots, same).tolist() == [[5, 1, 4, 0]]
    assert beam.reorder_rows([state], slots[:0], same[:0]).shape == (0, 4)


def test_reorder_flags_bad_indices_and_copies_nothing_for_them(cuda):
    state = torch.randn((1, 4, 8), device=cuda)
    keep = state.clone()
    slots = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=cuda)
    for parents, s in (([[0, 3, 1]], slots), ([[0, -1, 1]], slots),
                       ([[1, 1, 2]], torch.tensor([[9, 1, 2]], dtype=torch.int32, device=cuda))):
        beam.reorder_rows([state], s, torch.tensor(parents, dtype=torch.int32, device=cuda))
        with pytest.raises(_capi.DeviceFault):
            _capi.check_device()
        assert torch.equal(state, keep)


def test_reorder_refusals(cuda):
    state = torch.zeros((1, 4, 8), device=cuda)
    slots = torch.zeros((1, 3), dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError):
        beam.reorder_rows([state], slots, slots[:, :2].contiguous())
    with pytest.raises(TypeError):
        beam.reorder_rows([state], slots.long(), slots)
    with pytest.raises(ValueError):
        beam.reorder_rows([torch.zeros((4, 2, 8), device=cuda).transpose(0, 1)], slots, slots)
    with pytest.raises(ValueError):
        beam.reorder_rows([state] * 5, slots, slots)
    with pytest.raises(ValueError):
        beam.reorder_rows([state, torch.zeros((1, 5, 8), device=cuda)], slots, slots)
    with pytest.raises(_capi.ShellcacheError):
        beam.reorder_rows([torch.zeros((1, 4, 3), device=cuda)], slots, slots)
