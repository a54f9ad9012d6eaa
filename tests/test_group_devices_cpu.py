"""The group-decode operators' checks of their tensors (no GPU here: the tensors only say that
they are on one, and the launch is a recorder)."""

import pytest
import torch

from shellsmith_b200 import beam, paged, rotary


class OnDevice(torch.Tensor):
    """A CPU tensor that names a GPU as its device."""
    __torch_function__ = torch._C._disabled_torch_function_impl

    is_cuda = True
    index = 0

    def get_device(self):
        return self.index

    def new_empty(self, *args, **kw):
        return on(torch.Tensor.new_empty(self, *args, **kw), self.index)


def on(t, index=0):
    t = t.as_subclass(OnDevice)
    t.index = index
    return t


@pytest.fixture
def launched(monkeypatch):
    calls = []
    for module, name in ((rotary, "_append"), (beam, "_select"), (beam, "_reorder"),
                         (paged, "_shared_prefix")):
        monkeypatch.setattr(module, name, lambda *args, n=name: calls.append(n))
    for module in (rotary, beam, paged):
        monkeypatch.setattr(module, "fast", None)
        monkeypatch.setattr(module, "stream_of", lambda t: 0)
    return calls


def _bf(*shape):
    return on(torch.zeros(shape, dtype=torch.bfloat16))


def _plan(cls, *args, **kw):
    plan = cls(*args, device="cpu", **kw)
    plan.device_index = 0
    return plan


def test_rotary_takes_subclasses_of_tensor(launched):
    """A torch.nn.Parameter, say: the compiled caller takes it, and so does the wrapper."""
    plan = _plan(rotary.RotaryPlan, 64)
    pos = on(torch.zeros((1, 4), dtype=torch.int32))
    rotary.rotary(_bf(4, 2, 64), _bf(4, 1, 64), pos, plan)
    assert launched == ["_append"]
    for bad in (_bf(4, 2, 128)[..., ::2], _bf(4, 2, 32), _bf(4, 64)):
        with pytest.raises(ValueError):
            rotary.rotary(bad, _bf(4, 1, 64), pos, plan)
    with pytest.raises(TypeError):
        rotary.rotary(on(torch.zeros((4, 2, 64))), _bf(4, 1, 64), pos, plan)
    assert launched == ["_append"]


def _each_on_another(call, operands, launched):
    """call(**operands) launches; with any one operand on GPU 1 it raises and does not."""
    call(**operands)
    assert len(launched) == 1
    for name in operands:
        moved = dict(operands)
        t = moved[name]
        moved[name] = [on(t[0].clone(), 1)] if isinstance(t, list) else on(t.clone(), 1)
        with pytest.raises(ValueError, match="is on|are on"):
            call(**moved)
        assert len(launched) == 1, name


@pytest.mark.parametrize("append", [False, True])
def test_rotary(launched, append):
    plan = _plan(rotary.RotaryPlan, 64)
    operands = dict(q=_bf(4, 2, 64), k=_bf(4, 1, 64),
                    positions=on(torch.zeros((1, 4), dtype=torch.int32)),
                    q_weight=_bf(64), k_weight=_bf(64))
    if not append:
        _each_on_another(lambda **kw: rotary.rotary(plan=plan, **kw), operands, launched)
        return
    operands.update(v=_bf(4, 1, 64), kv_pool=_bf(2, 1, 2, 16, 64),
                    slot_mapping=on(torch.zeros(4, dtype=torch.int64)), out=_bf(4, 2, 64))
    _each_on_another(lambda **kw: rotary.rotary_append(plan=plan, **kw), operands, launched)


def test_beam_select(launched, monkeypatch):
    monkeypatch.setattr(beam, "_workspace", lambda *a: 256)
    operands = dict(logits=_bf(2, 3, 50), scores=on(torch.zeros((2, 3))),
                    finished=on(torch.zeros((2, 3), dtype=torch.bool)))
    _each_on_another(lambda **kw: beam.beam_select(n=4, **kw), operands, launched)


def test_reorder_rows(launched):
    ids = torch.zeros((1, 3), dtype=torch.int32)
    operands = dict(pools=[_bf(1, 4, 8)], slots=on(ids), parents=on(ids.clone()))
    _each_on_another(lambda **kw: beam.reorder_rows(**kw), operands, launched)


@pytest.mark.parametrize("rows", [[0, 1], [0]])
def test_shared_prefix_attention(launched, monkeypatch, rows):
    monkeypatch.setattr(paged._capi, "call", lambda *a: launched.append(a[0]))
    monkeypatch.setattr(paged, "sm_count", lambda d: 148)
    groups = _plan(paged.PrefixGroups, [(rows, 32)], 2, 4, 2, 64, sms=148)
    assert groups.ntiles == (len(rows) > 1)
    operands = dict(q=_bf(2, 4, 64), kv_pool=_bf(8, 2, 2, 16, 64),
                    block_table=on(torch.zeros((2, 4), dtype=torch.int32)),
                    ctx_len=on(torch.zeros(2, dtype=torch.int32)), out=_bf(2, 4, 64),
                    lse_out=on(torch.zeros(8)))
    ws = paged.SharedPrefixWorkspace("cpu")
    ws.device_index = 0
    call = lambda **kw: paged.shared_prefix_attention(scale=0.1, groups=groups, workspace=ws,  # noqa: E731
                                                      **kw)
    _each_on_another(call, operands, launched)
    other = paged.SharedPrefixWorkspace("cpu")
    other.device_index = 1
    if groups.ntiles:
        with pytest.raises(ValueError):
            paged.shared_prefix_attention(scale=0.1, groups=groups, workspace=other, **operands)
        assert len(launched) == 1


def test_beam_select_refuses_numbers_that_do_not_fit(launched, monkeypatch):
    """2^32 + 2 tokens from the pad token's place would be token 2 in the C call."""
    monkeypatch.setattr(beam, "_workspace", lambda *a: 256)
    x, s = _bf(2, 3, 50), on(torch.zeros((2, 3)))
    done = on(torch.zeros((2, 3), dtype=torch.bool))
    for pad in (2 ** 32 + 2, 2 ** 31, -2 ** 31 - 1):
        with pytest.raises(ValueError):
            beam.beam_select(x, s, 4, finished=done, pad_token=pad)
    for n in (2 ** 32 + 4, -1, -2 ** 40):
        with pytest.raises(ValueError):
            beam.beam_select(x, s, n)
    for n in (4.0, "4", None):
        with pytest.raises(TypeError):
            beam.beam_select(x, s, n)
    assert not launched


@pytest.mark.parametrize("bits", [8, 16])
def test_rotary_append_refuses_another_out(launched, monkeypatch, bits):
    """Of 8-bit pools too, whose q is copied to out: one token would be spread over a larger
    one, and rounded or widened into another type."""
    monkeypatch.setattr(paged, "kv_append", lambda *a: launched.append("kv_append"))
    plan = _plan(rotary.RotaryPlan, 128)
    pool = on(torch.zeros((4, 1, 34 * 128), dtype=torch.uint8)) if bits == 8 else _bf(4, 1, 2, 16, 128)
    args = (_bf(1, 2, 128), _bf(1, 1, 128), _bf(1, 1, 128), on(torch.zeros((1, 1), dtype=torch.int32)),
            plan, pool, on(torch.zeros(1, dtype=torch.int64)))
    for out in (_bf(5, 2, 128), _bf(1, 2, 64), _bf(2, 128), _bf(1, 128, 2).transpose(1, 2),
                on(torch.zeros((1, 2, 128)))):
        with pytest.raises((ValueError, TypeError)):
            rotary.rotary_append(*args, out=out)
        assert not launched
    out = _bf(1, 2, 128)
    assert rotary.rotary_append(*args, out=out) is out and launched


@pytest.mark.parametrize("first", [0, 1, 3, 8])
def test_rotary_append_of_one_token_off_a_boundary_to_8_bit_pages(launched, monkeypatch, first):
    """One token's view of v is contiguous wherever it starts; the append wants 16 bytes."""
    taken = []
    monkeypatch.setattr(paged, "kv_append", lambda k, v, *a: taken.append(v))
    plan = _plan(rotary.RotaryPlan, 128)
    v = on(torch.arange(140, dtype=torch.bfloat16)[first:first + 128].view(1, 1, 128))
    rotary.rotary_append(_bf(1, 2, 128), _bf(1, 1, 128), v, on(torch.zeros((1, 1), dtype=torch.int32)),
                         plan, on(torch.zeros((4, 1, 34 * 128), dtype=torch.uint8)),
                         on(torch.zeros(1, dtype=torch.int64)))
    assert taken[0].is_contiguous() and taken[0].data_ptr() % 16 == 0
    assert torch.equal(taken[0].as_subclass(torch.Tensor), v.as_subclass(torch.Tensor))


@pytest.mark.parametrize("pages", [8 * 1023, 8 * 1024, 8 * 1500, 20_000])
def test_prefix_in_more_splits_than_the_merge_takes(launched, monkeypatch, pages):
    """Split sizes of the caller's own that leave no part to the sequences' own pages: the plan
    ends all the same, and the entry point says what is wrong."""
    monkeypatch.setattr(paged, "most_splits", lambda *a: 4096)
    groups = _plan(paged.PrefixGroups, [([0, 1], 16 * pages)], 2, 4, 2, 64, sms=148,
                   pages_per_split=8)
    paged.shared_prefix_attention(_bf(2, 4, 64), _bf(8, 2, 2, 16, 64),
                                  on(torch.zeros((2, pages), dtype=torch.int32)),
                                  on(torch.zeros(2, dtype=torch.int32)), 0.1, groups)
    assert launched == ["_shared_prefix"]
