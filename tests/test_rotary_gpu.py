"""Rotary positions, q/k norm and KV append (rotary.py) on the GPU vs the formula in 64 bits.

Bars. The result is one rounding of an fp32 value to bf16, whose 8 significant bits put a
nearest value at most 2^-8 of the size away, plus the fp32 steps before it (a product sum
of two terms, the norm's mean and rsqrt: under 1e-6 of a head's largest value, here below
8), so rtol 2^-8 * 1.01 and atol 1e-5. The angle is reduced in double, so large positions keep the same bars. Pool bytes that no slot
names, and v, are bit-exact.
"""

import numpy as np
import pytest
import torch

from oracle import attention as oatt
from shellsmith_b200 import _capi, paged, rotary

pytestmark = pytest.mark.gpu

RTOL, ATOL = 2.0 ** -8 * 1.01, 1e-5


def _axes(sections, interleaved):
    half, A = sum(sections), len(sections)
    out = []
    for i in range(half):
        if interleaved:
            a = i % A
            out.append(a if i // A < sections[a] else 0)
        else:
            out.append(int(np.searchsorted(np.cumsum(sections), i, side="right")))
    return out


def _reference(x, weight, pos, sections, interleaved, base, rot, eps=1e-6):
    x = x.double().cpu().numpy()
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * weight.double().cpu().numpy()
    half = rot // 2
    freq = base ** (-np.arange(half) / half)
    t = pos.cpu().numpy().astype(np.float64)[_axes(sections, interleaved)].T * freq  # [n, half]
    c, s = np.cos(t)[:, None], np.sin(t)[:, None]
    y = x.copy()
    a, b = x[..., :half], x[..., half:rot]
    y[..., :half], y[..., half:rot] = a * c - b * s, b * c + a * s
    return y


def _close(got, want):
    np.testing.assert_allclose(got.double().cpu().numpy(), want, rtol=RTOL, atol=ATOL)


CASES = [  # tokens, Hq, Hkv, D, rot, sections, interleaved, norm, first position
    (1, 16, 2, 256, 64, (11, 11, 10), True, True, 0),
    (8, 16, 2, 256, 64, (12, 10, 10), False, True, 16384),
    (33, 24, 8, 128, 128, (64,), False, False, 1000),
    (5, 3, 1, 64, 16, (4, 2, 2), True, True, 262000),
    (17, 4, 4, 64, 64, (16, 8, 8), True, False, 1_000_000),
    (1025, 6, 2, 128, 32, (16,), False, True, 7),
    (2050, 8, 1, 256, 256, (43, 43, 42), True, True, 99),
]


@pytest.mark.parametrize("n,hq,hkv,D,rot,sections,inter,norm,start", CASES)
@pytest.mark.parametrize("layout", ["dense", "views", "odd"])
def test_rotary_matches_formula(cuda, n, hq, hkv, D, rot, sections, inter, norm, start, layout):
    if layout == "dense":
        q, k = torch.randn((n, hq, D), device=cuda), torch.randn((n, hkv, D), device=cuda)
        q, k = q.to(torch.bfloat16), k.to(torch.bfloat16)
    elif layout == "views":   # q beside its gate, k beside v
        q = torch.randn((n, hq, 2 * D), device=cuda).to(torch.bfloat16)[..., :D]
        k = torch.randn((n, 2 * hkv, D), device=cuda).to(torch.bfloat16)[:, hkv:]
    else:                     # rows that start at odd elements, heads before tokens
        q = torch.randn((hq, n, D + 3), device=cuda).to(torch.bfloat16)[..., 3:].transpose(0, 1)
        k = torch.randn((n, hkv, D + 1), device=cuda).to(torch.bfloat16)[..., 1:]
    pos = torch.stack([start + torch.arange(n) * (1 if a == 0 else 0) + torch.randint(0, 40, (n,)) * (a > 0)
                       for a in range(len(sections))]).to(torch.int32).to(cuda)
    qw = (1 + 0.2 * torch.randn(D, device=cuda)).to(torch.bfloat16) if norm else None
    kw = (1 + 0.2 * torch.randn(D, device=cuda)).to(torch.bfloat16) if norm else None
    plan = rotary.RotaryPlan(D, rot, base=10000.0, sections=sections, interleaved=inter, device=cuda)
    qo, ko = rotary.rotary(q, k, pos, plan, q_weight=qw, k_weight=kw)
    assert qo.is_contiguous() and ko.is_contiguous()
    _close(qo, _reference(q, qw, pos, sections, inter, 10000.0, rot))
    _close(ko, _reference(k, kw, pos, sections, inter, 10000.0, rot))


@pytest.mark.parametrize("n,hkv,D,P", [(1, 2, 256, 16), (40, 2, 256, 16), (37, 8, 128, 8),
                                       (1100, 1, 64, 32)])
def test_rotary_append_writes_the_pool(cuda, n, hkv, D, P):
    rng = np.random.default_rng(n)
    pages = -(-n // P) + 3
    slots = rng.permutation(pages * P)[:n].astype(np.int64)
    if n > 5:
        slots[[2, 5]] = -1
    q = torch.randn((n, 2 * hkv, D), device=cuda).to(torch.bfloat16)
    kv = torch.randn((n, 2 * hkv, D), device=cuda).to(torch.bfloat16)
    k, v = kv[:, :hkv], kv[:, hkv:]
    pos = torch.arange(n, dtype=torch.int32, device=cuda) + 50
    plan = rotary.RotaryPlan(D, device=cuda)
    pool = torch.randn((pages, hkv, 2, P, D), device=cuda).to(torch.bfloat16)
    want = pool.clone()
    slot_t = torch.from_numpy(slots).to(cuda)
    out = rotary.rotary_append(q, k, v, pos, plan, pool, slot_t)
    qo, ko = rotary.rotary(q, k, pos[None], plan)
    assert torch.equal(out, qo)
    paged.kv_append(ko, v.contiguous(), want, slot_t)  # the same bits through the two-launch path
    assert torch.equal(pool, want)
    _capi.check_device()


def test_rotary_append_to_8bit_pool_equals_two_calls(cuda):
    n, hkv, D = 21, 2, 128
    q = torch.randn((n, 8, D), device=cuda).to(torch.bfloat16)
    kv = torch.randn((n, 2 * hkv, D), device=cuda).to(torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int32, device=cuda)
    plan = rotary.RotaryPlan(D, 64, device=cuda)
    slots = torch.randperm(4 * 16, device=cuda)[:n]
    a, b = paged.new_pool_q8(4, hkv, D, device=cuda), paged.new_pool_q8(4, hkv, D, device=cuda)
    a.zero_(), b.zero_()
    out = rotary.rotary_append(q, kv[:, :hkv], kv[:, hkv:], pos, plan, a, slots)
    qo, ko = rotary.rotary(q, kv[:, :hkv], pos, plan)
    paged.kv_append(ko, kv[:, hkv:].contiguous(), b, slots)
    assert torch.equal(out, qo) and torch.equal(a, b)


def test_rotary_inverse_turns_back(cuda):
    """Turning by -position undoes a turn (a rotation keeps lengths): two bf16 roundings."""
    n, D = 64, 128
    x = torch.randn((n, 4, D), device=cuda).to(torch.bfloat16)
    pos = torch.randint(0, 5000, (n,), device=cuda, dtype=torch.int32)
    plan = rotary.RotaryPlan(D, device=cuda)
    y, _ = rotary.rotary(x, x[:, :1], pos, plan)
    z, _ = rotary.rotary(y, y[:, :1], -pos, plan)
    # The first rounding moves the pair by at most 2^-8 of its length, which a turn keeps;
    # the second moves each element by 2^-8 of its own size.
    pair = (x[..., :D // 2].float() ** 2 + x[..., D // 2:].float() ** 2).sqrt().repeat(1, 1, 2)
    assert ((z.float() - x.float()).abs() <= 2.0 ** -8 * 2.02 * pair + 1e-5).all()


def test_empty_and_bad_slots(cuda):
    plan = rotary.RotaryPlan(64, device=cuda)
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device=cuda)
    pos = torch.empty((0,), dtype=torch.int32, device=cuda)
    pool = torch.zeros((2, 1, 2, 16, 64), dtype=torch.bfloat16, device=cuda)
    none = torch.empty((0,), dtype=torch.int64, device=cuda)
    assert rotary.rotary_append(q, q[:, :1], q[:, :1], pos, plan, pool, none).shape == q.shape
    x = torch.ones((1, 1, 64), dtype=torch.bfloat16, device=cuda)
    rotary.rotary_append(x, x, x, torch.zeros(1, dtype=torch.int32, device=cuda), plan, pool,
                         torch.tensor([2 * 16], device=cuda))
    with pytest.raises(_capi.DeviceFault):
        _capi.check_device()
    assert not pool.any()


def test_refusals(cuda):
    bf = dict(dtype=torch.bfloat16, device=cuda)
    q, pos = torch.zeros((4, 2, 128), **bf), torch.zeros(4, dtype=torch.int32, device=cuda)
    plan = rotary.RotaryPlan(128, device=cuda)
    with pytest.raises(ValueError):
        rotary.RotaryPlan(96, device=cuda)
    with pytest.raises(ValueError):
        rotary.RotaryPlan(128, 24, device=cuda)
    with pytest.raises(ValueError):
        rotary.RotaryPlan(128, sections=(30, 30), device=cuda)
    with pytest.raises(ValueError):
        rotary.RotaryPlan(128, inv_freq=[1.0], device=cuda)
    with pytest.raises(TypeError):
        rotary.rotary(q.float(), q, pos, plan)
    with pytest.raises(ValueError):
        rotary.rotary(q[..., :64], q, pos, plan)
    with pytest.raises(ValueError):
        rotary.rotary(q, q[:3], pos, plan)
    with pytest.raises(ValueError):
        rotary.rotary(q, q, pos[:3], plan)
    with pytest.raises(ValueError):
        rotary.rotary(q, q, pos.long(), plan)
    with pytest.raises(ValueError):
        rotary.rotary(q.transpose(1, 2).contiguous().transpose(1, 2), q, pos, plan)
    with pytest.raises(ValueError):
        rotary.rotary(q, q, pos, plan, q_weight=torch.zeros(64, **bf))
    pool = torch.zeros((2, 2, 2, 16, 128), **bf)
    slots = torch.zeros(4, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError):
        rotary.rotary_append(q, q, q, pos, plan, pool, slots[:2])
    with pytest.raises(ValueError):
        rotary.rotary_append(q, q[:, :1], q[:, :1], pos, plan, pool, slots)
    with pytest.raises(ValueError):
        rotary.rotary_append(q.cpu(), q, q, pos, plan, pool, slots)


def test_pool_layout_matches_the_oracle(cuda):
    """Position 0 turns nothing: the pool holds k and v themselves, in the oracle's layout."""
    n, hkv, P, D = 9, 2, 16, 256
    k = torch.randn((n, hkv, D), device=cuda).to(torch.bfloat16)
    pos = torch.zeros(n, dtype=torch.int32, device=cuda)
    pool = torch.zeros((2, hkv, 2, P, D), dtype=torch.bfloat16, device=cuda)
    slots = np.arange(n, dtype=np.int64) + 11
    rotary.rotary_append(k, k, -k, pos, rotary.RotaryPlan(D, device=cuda), pool,
                         torch.from_numpy(slots).to(cuda))
    want = np.zeros(pool.numel(), np.uint16)
    bits = lambda t: t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)  # noqa: E731
    oatt.pool_write(want, slots, bits(k), bits(-k), hkv, P, D)
    assert np.array_equal(bits(pool).reshape(-1), want)
