"""Shared-prefix decode attention (paged.shared_prefix_attention) at its edges: short tails
over many units of work, infinities in the cache, long sequences without a group. Cases, the
64-bit reference and the bars are those of the operator's own tests."""

import pytest
from test_shared_prefix_gpu import _case, _check

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
