"""Selections whose candidate lists overflow (beam.beam_select): long runs of equal large
logits, sparse masks, and many continuations asked for (n + 1 entries of each of a segment's
eight warps pass the list). They take the pass that goes over the segment in index order.

One beam with score 0: its order is that of its logits, equal ones by the lower token. All
logits here are bf16 values, whose differences (2^-8 of their size) no fp32 score merges, so
the tokens are exact; scores within the bar of the selection's own tests (2e-5).
"""

import pytest
import torch

from shellsmith_b200 import _capi, beam

pytestmark = pytest.mark.gpu

TOL = 2e-5


def _exact(logits, n):
    """Rows [R, V] of one-beam groups, against a stable sort."""
    R, V = logits.shape
    got, parents, tokens = beam.beam_select(logits[:, None].contiguous(),
                                            torch.zeros((R, 1), device=logits.device), n)
    _capi.check_device()
    x = logits.double()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :n]
    assert not parents.any()
    assert torch.equal(tokens.long(), order)
    want = torch.log_softmax(x, -1).gather(1, order)
    live = want > -float("inf")
    assert torch.equal(torch.isneginf(got), ~live)
    assert (got.double() - want)[live].abs().max() <= TOL


def _rows(kind, R, V, cuda):
    at = torch.arange(V, device=cuda)
    if kind == "constant":
        x = torch.full((R, V), 1.5, device=cuda)
    elif kind == "two values":
        x = torch.where(torch.rand((R, V), device=cuda) < 0.5, 1.5, 0.25)
    elif kind == "rising runs":      # each run of equal values above the last
        x = (at // 700).float().mul(0.03125).expand(R, V).contiguous()
    elif kind == "sparse":           # a masked vocabulary with one value left here and there
        x = torch.where(torch.rand((R, V), device=cuda) < 0.03, 2.0, -float("inf"))
    else:                            # what a model gives
        x = torch.randn((R, V), device=cuda) * 2.5
    return x.to(torch.bfloat16).float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [16, 44, 64])
@pytest.mark.parametrize("kind", ["constant", "two values", "rising runs", "sparse", "normal"])
def test_overflowing_lists(cuda, dtype, n, kind):
    for R, V in ((1, 70003), (6, 40001), (600, 9000)):
        x = _rows(kind, R, V, cuda).to(dtype)
        for _ in range(3):
            _exact(x, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("left", [129, 130, 131])
def test_tile_after_a_list_that_is_just_not_cut(cuda, dtype, left):
    """n = 64: a segment whose first tile (256 granules of 16 bytes) leaves 129 to 131 logits,
    one a granule and 65 in each of the first two blocks of 128, before tiles of equal lower
    ones. 130 entries are not cut yet, and the next tile appends a whole tile's."""
    per = 16 // dtype.itemsize
    V = 60 * 256 * per
    x = torch.full((V,), 0.5, device=cuda)
    x[:256 * per] = -float("inf")
    block = torch.arange(128, device=cuda) * per
    first = torch.cat([block[:65], block[:65] + 128 * per, block[65:70]])[:left]
    x[first] = 2.0 + torch.arange(left, device=cuda) % 7 * 0.125
    for R in (1, 5, 700):
        _exact(x.to(dtype).expand(R, V).contiguous(), 64)


def test_reorder_without_pools_flags_nothing(cuda):
    """The new slots alone: no row is out of range where there is none."""
    slots = torch.tensor([[4, 1, 0, 5]], dtype=torch.int32, device=cuda)
    parents = torch.tensor([[2, 2, 0, 2]], dtype=torch.int32, device=cuda)
    _capi.device_status()
    assert beam.reorder_rows([], slots, parents).tolist() == [[0, 1, 4, 5]]
    assert beam.reorder_rows((), slots, parents).tolist() == [[0, 1, 4, 5]]
    _capi.check_device()
    with pytest.raises(_capi.DeviceFault):
        beam.reorder_rows([], slots, parents + 9)
        _capi.check_device()
    with pytest.raises(_capi.ShellcacheError):
        beam.reorder_rows([torch.empty((2, 0, 8), device=cuda)], slots, parents)
