"""Selections on the GPU, looked at one successor at a time: each that is returned is a successor, with the score that it has, in its place; and it is the same whenever it is made."""
import ctypes as C

import numpy as np
import pytest
import torch

from koboldcpp_b200.lib import check, lib
from test_gpu_beam import Select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,beams,vocab,keep", [(64, 1, 1, 1), (64, 2, 3, 5), (40, 4, 40, 8), (16, 8, 600, 16), (8, 16, 1300, 64)])
def test_few_candidates_again_and_again(requests, beams, vocab, keep):
    """Lists so short that some warps are through them before others have begun: hundreds of calls, all with the first one's results."""
    s = Select(requests, beams, vocab, keep, seed=vocab)
    s.run().verify()
    first = [t.clone() for t in s.to]
    for _ in range(300):
        for t in s.to:
            t.fill_(77)
        check(lib().b200_op_beam_select(C.byref(s.args), s.ws.data_ptr(), s.ws.numel(), None))
        assert all(torch.equal(a, b) for a, b in zip(s.to, first))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 2000, 70000])
def test_scores_and_logits_of_plus_infinity(kind, vocab):
    """A beam of score +inf comes before all others; where its row has logits of +inf, these are its only successors."""
    s = Select(3, 4, vocab, 12, kind, seed=vocab)
    s.score[[1, 6]] = np.inf
    s.logits[1, [3, 30, vocab - 1]] = np.inf
    s.logits[2, 5] = np.inf
    s.run()
    beam, token, score, slot = (s.to[i][:-1].cpu().numpy().reshape(3, 12) for i in (1, 2, 0, 3))
    assert beam[0, :4].tolist() == [1, 1, 1, 2] and token[0, :4].tolist() == [3, 30, vocab - 1, 5] and (score[0, :3] == np.inf).all()
    assert score[0, 3] == s.score[2] and (np.diff(score[0, 3:]) <= 0).all() and (beam[0, 4:] % 3 == 0).all()
    assert (beam[1] == 2).all() and token[1].tolist() == list(range(12)) and (score[1] == np.inf).all()  # (equal ones by their place)
    assert np.isfinite(score[2]).all() and np.array_equal(slot, np.take_along_axis(s.slot.reshape(3, 4), beam, 1))
