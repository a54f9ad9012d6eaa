"""Shared-prefix decode attention (paged.shared_prefix_attention) on the GPU vs softmax
attention in 64 bits.

Bar, element by element. The probabilities enter the P V product rounded to bf16 (at most
2^-8 of each), their sum does not: |error| <= 2^-8 sum_j p_j |v_j|, plus 2^-8 |out| for
the output's own rounding. fp32 scores (256 products, |s| < 64) are off by less than 1e-4,
which moves p and so the output by that share of sum_j p_j |v_j| again; twice that for the
parts' weights. Pool rows that no sequence attends to hold NaN.
"""

import math

import numpy as np
import pytest
import torch

from oracle import attention as oatt
from shellsmith_b200 import _capi, paged

pytestmark = pytest.mark.gpu
P = paged.PAGE_SIZE


def _case(cuda, groups, tails, hq, hkv, D, seed=0, single=()):
    """groups: [(rows, prefix tokens)]; tails: tokens past the prefix by row (None: no
    context at all); single: context lengths of ungrouped rows, appended at the end."""
    rng = np.random.default_rng(seed)
    B = sum(r for r, _ in groups) + len(single)
    prefix = [p for r, p in groups for _ in range(r)] + [0] * len(single)
    ctx = np.array([0 if t is None else p + t for p, t in zip(prefix, list(tails) + list(single))])
    width = max(1, max(-(-max(p, int(c)) // P) for p, c in zip(prefix, ctx)))
    free = iter(rng.permutation(4 * B + 4 + sum(-(-int(c) // P) for c in ctx)
                                + sum(p // P for _, p in groups)).tolist())
    table, plan, b = np.zeros((B, width), np.int32), [], 0
    for r, p in groups:
        shared = [next(free) for _ in range(p // P)]
        plan.append((range(b, b + r), p))
        for _ in range(r):
            table[b, :len(shared)] = shared
            b += 1
    for i in range(B):
        for j in range(prefix[i] // P, -(-int(ctx[i]) // P)):
            table[i, j] = next(free)
    pages = 8 * B + 8 + int(table.max())
    pool = torch.full((pages, hkv, 2, P, D), float("nan"), dtype=torch.bfloat16, device=cuda)
    read = np.zeros((pages, P), bool)
    for i in range(B):
        for t in range(int(ctx[i])):
            read[table[i, t // P], t % P] = True
    at = torch.from_numpy(np.flatnonzero(read.reshape(-1))).to(cuda)
    kv = torch.randn((2, at.numel(), hkv, D), device=cuda).to(torch.bfloat16)
    if at.numel():
        paged.kv_append(kv[0], kv[1], pool, at)
    q = (2 * torch.randn((B, hq, D), device=cuda)).to(torch.bfloat16)
    return q, pool, table, ctx, plan


def _expect(q, pool, table, ctx, scale):
    pn, qn = pool.float().cpu().numpy(), q.double().cpu().numpy()
    B, hq, D = qn.shape
    hkv = pn.shape[1]
    out, lse, mass = np.zeros((B, hq, D)), np.full((B, hq), -np.inf), np.zeros((B, hq, D))
    for b in range(B):
        if ctx[b] == 0:
            continue
        k, v = oatt.pool_read_pages(pn, table[b], int(ctx[b]), hkv, P, D)
        k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)     # [L, Hkv, D]
        for h in range(hq):
            s = scale * (k[:, h // (hq // hkv)] @ qn[b, h])
            m = s.max()
            e = np.exp(s - m)
            p = e / e.sum()
            out[b, h] = p @ v[:, h // (hq // hkv)]
            mass[b, h] = p @ np.abs(v[:, h // (hq // hkv)])
            lse[b, h] = m + np.log(e.sum())
    return out, lse, mass


def _run(cuda, case, scale, sms=None, hint=True, **kw):
    q, pool, table, ctx, plan = case
    B, hq, D = q.shape
    groups = paged.PrefixGroups(plan, B, hq, pool.shape[1], D, device=cuda, sms=sms)
    lse = torch.empty(B * hq, dtype=torch.float32, device=cuda)
    own = [-(-int(c) // P) - (min(p // P, int(c) // P)) for c, p in
           zip(ctx, [p for r, p in plan for _ in r] + [0] * B)]
    if hint:
        kw.update(max_suffix_pages=max(1, max(own)), total_suffix_pages=sum(own))
    out = paged.shared_prefix_attention(q, pool, torch.from_numpy(table).to(cuda),
                                        torch.from_numpy(ctx.astype(np.int32)).to(cuda), scale,
                                        groups, lse_out=lse, **kw)
    _capi.check_device()
    return out, lse.view(B, hq)


def _check(cuda, case, scale=None, **kw):
    q, pool, table, ctx, _ = case
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out, lse = _run(cuda, case, scale, **kw)
    want, want_lse, mass = _expect(q, pool, table, ctx, scale)
    got = out.double().cpu().numpy()
    tol = (2.0 ** -8 + 3e-4) * mass + 2.0 ** -8 * 1.01 * np.abs(want) + 1e-6
    worst = np.max(np.abs(got - want) / tol)
    assert np.isfinite(got).all() and worst <= 1, worst
    np.testing.assert_allclose(lse.cpu().numpy(), want_lse, atol=1e-3)
    return out


SHAPES = [(16, 2, 256), (24, 8, 128), (8, 8, 64), (12, 1, 256), (6, 1, 128), (64, 1, 64), (40, 1, 128)]


@pytest.mark.parametrize("hq,hkv,D", SHAPES)
@pytest.mark.parametrize("sms", [1, 148])
def test_matches_64_bits(cuda, hq, hkv, D, sms):
    """Sizes around pages, tiles (64 / 128 tokens) and rings of stages, several groups."""
    groups = [(2, 16), (5, 48), (3, 64), (2, 80), (3, 21 * 16), (4, 50 * 16)]
    tails = [1, 15, 16, 17, 0, 3, 200, 1, 2, 31, 64, 5, 1, 130, 1, 1, 33, 7, 16]
    case = _case(cuda, groups, tails, hq, hkv, D, seed=hq + D, single=[1, 100, 0])
    _check(cuda, case, sms=sms)


@pytest.mark.parametrize("hq,hkv,D,rows", [(16, 2, 256, 33), (4, 4, 64, 130), (12, 4, 128, 43),
                                           (128, 1, 128, 3)])
def test_groups_larger_than_a_tile(cuda, hq, hkv, D, rows):
    case = _case(cuda, [(rows, 33 * 16)], [1 + (7 * i) % 40 for i in range(rows)], hq, hkv, D)
    _check(cuda, case)
    _check(cuda, case, hint=False)


def test_long_prefix_many_splits(cuda):
    case = _case(cuda, [(4, 6000), (4, 2512)], [1, 700, 40, 9, 16, 16, 100, 3], 16, 2, 256, seed=4)
    a = _check(cuda, case)
    b = _check(cuda, case, sms=7)
    assert (a.float() - b.float()).abs().max() < 0.05


def test_contexts_that_end_inside_the_prefix(cuda):
    """Members whose context is shorter than the shared pages, or empty."""
    for sms in (1, 148):
        case = _case(cuda, [(7, 160), (3, 320)], [4, -1, -16, -100, -159, None, 1, None, -310, -305],
                     16, 2, 256, seed=2)
        out = _check(cuda, case, sms=sms)
        assert not out[5].any() and not out[7].any()


def test_no_member_reaches_the_prefix(cuda):
    case = _case(cuda, [(3, 160)], [None, None, None], 16, 2, 256)
    out, lse = _run(cuda, case, 0.1)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.4])
def test_scales(cuda, scale):
    """A zero scale averages the values, a negative one prefers the smallest products, a
    large one makes the running maximum grow from tile to tile."""
    _check(cuda, _case(cuda, [(3, 40 * 16)], [1, 30, 17], 8, 2, 128, seed=5), scale=scale)


def test_growing_scores_rescale(cuda):
    """Keys that grow along the prefix: the reference maximum moves in every tile."""
    case = _case(cuda, [(2, 60 * 16)], [1, 18], 16, 2, 256, seed=6)
    q, pool, table, ctx, plan = case
    pages = torch.from_numpy(table[0, :60].astype(np.int64)).to(cuda)
    grow = torch.linspace(0.1, 6.0, 60, device=cuda)[:, None, None, None]
    pool[pages, :, 0] = (pool[pages, :, 0].float() * grow).to(torch.bfloat16)
    _check(cuda, case)
    pool[pages, :, 0] = pool[pages.flip(0), :, 0].clone()  # and shrink
    _check(cuda, case)


def test_equals_plain_decode_without_groups(cuda):
    case = _case(cuda, [], [], 16, 2, 256, single=[5, 100, 33])
    q, pool, table, ctx, _ = case
    groups = paged.PrefixGroups([([0], 16), ([1, 2], 15)], 3, 16, 2, 256, device=cuda)
    assert groups.ntiles == 0
    t, c = torch.from_numpy(table).to(cuda), torch.from_numpy(ctx.astype(np.int32)).to(cuda)
    a = paged.shared_prefix_attention(q, pool, t, c, 0.06, groups)
    assert torch.equal(a, paged.paged_decode_attention(q, pool, t, c, 0.06))


def test_side_stream_workspace_and_repeats(cuda):
    """Calls back to back on another stream reuse one workspace; the result repeats bit for bit."""
    case = _case(cuda, [(8, 1600)], [1 + 9 * i for i in range(8)], 16, 2, 256, seed=9)
    ws = paged.SharedPrefixWorkspace(cuda)
    first, _ = _run(cuda, case, 0.0625)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [_run(cuda, case, 0.0625, workspace=ws)[0] for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, first) for o in outs)


def test_bad_pages_are_flagged(cuda):
    q, pool, table, ctx, plan = _case(cuda, [(2, 160)], [1, 1], 16, 2, 256)
    table = table.copy()
    table[:, 4] = pool.shape[0]
    pool.zero_()
    groups = paged.PrefixGroups(plan, 2, 16, 2, 256, device=cuda)
    out = paged.shared_prefix_attention(q, pool, torch.from_numpy(table).to(cuda),
                                        torch.from_numpy(ctx.astype(np.int32)).to(cuda), 0.1, groups)
    with pytest.raises(_capi.DeviceFault):
        _capi.check_device()
    assert torch.isfinite(out).all()


def test_refusals(cuda):
    q, pool, table, ctx, plan = _case(cuda, [(2, 160)], [1, 1], 16, 2, 256)
    t, c = torch.from_numpy(table).to(cuda), torch.from_numpy(ctx.astype(np.int32)).to(cuda)
    make = lambda groups, hq=16, hkv=2, D=256, B=2: paged.PrefixGroups(  # noqa: E731
        groups, B, hq, hkv, D, device=cuda)
    for bad in ([([0, 2], 16)], [([0, -1], 16)], [([0, 0], 16)], [([0, 1], 16), ([1], 16)],
                [([0, 1], -16)]):
        with pytest.raises(ValueError):
            make(bad)
    with pytest.raises(ValueError):
        make(plan, hq=130, hkv=1)
    with pytest.raises(ValueError):
        make(plan, D=96)
    groups = make(plan)
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(q[:1], pool, t, c, 0.1, groups)
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(q, pool, t[:, :9].contiguous(), c, 0.1, groups)
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(q, pool, t, c, 0.1, make(plan, hq=32))
    with pytest.raises(ValueError):
        paged.shared_prefix_attention(q, pool, t, c, 0.1, groups,
                                      lse_out=torch.empty(3, device=cuda))
    with pytest.raises(TypeError):
        paged.shared_prefix_attention(q.float(), pool, t, c, 0.1, groups)
    with pytest.raises(TypeError):
        paged.shared_prefix_attention(q, paged.new_pool_q8(4, 2, 256, device=cuda), t, c, 0.1, groups)
