"""What BeamSearch chooses, against the logits that it chose from.

Every step's logits, earlier scores and finished flags are recorded on their way into the
selection; the beams that go on have to be the best continuations in 64 bits, in order. The
scores' bar is the selection's own (2e-5, sizes below 2^6); a choice may only differ from the
64-bit order where two scores are closer than that.
"""

import numpy as np
import pytest
import torch
from test_group_decode_gpu import _cfg, _search

from shellsmith_b200.resident import ToyHybridModel

pytestmark = pytest.mark.gpu
TOL = 2e-5


@pytest.mark.parametrize("beams", [1, 4, 9])
@pytest.mark.parametrize("stops", [False, True])
def test_the_best_continuations_go_on(cuda, beams, stops):
    cfg = _cfg()
    model = ToyHybridModel(cfg, device=cuda)
    stop = None
    if stops:  # the token that the prompt's most likely continuation starts with
        _, probe = _search(cuda, cfg, model)
        probe.start([7, 8, 9], 1)
        stop = probe.beams[0].tokens[0]
    eng, search = _search(cuda, cfg, model, stop=stop)
    choose, seen = search._choose, []

    def record():
        old = [(list(b.tokens), b.finished) for b in search.beams]
        logits, scores = search._logits.double().cpu(), search._scores[0].double().cpu()
        choose()
        total = scores[:, None] + torch.log_softmax(logits, -1)
        for i, (_, finished) in enumerate(old):
            if finished:
                total[i] = -float("inf")
                total[i, stop] = scores[i]
        best = total.flatten().topk(beams).values
        got = []
        for b in search.beams:
            if b.finished and (b.tokens, True) in old:   # it stays what it was
                at = [o == (b.tokens, True) for o in old].index(True)
                got.append(float(scores[at]))
                assert b.score == got[-1]
            else:
                parents = [i for i, (t, f) in enumerate(old) if t == b.tokens[:-1] and not f]
                assert parents
                got.append(max(float(total[i, b.tokens[-1]]) for i in parents))
                assert b.finished == (b.tokens[-1] == stop)
            assert abs(b.score - got[-1]) <= TOL
        np.testing.assert_allclose(got, best.numpy(), rtol=0, atol=TOL)
        if beams == 1 and not old[0][1]:
            assert float(logits[0, search.beams[0].tokens[-1]]) == float(logits[0].max())
        seen.append(len(old))

    search._choose = record
    search.start([7, 8, 9], beams)
    for _ in range(8):
        if not search.step():
            break
    assert seen and (stops or len(seen) == 9)
    search.close()
