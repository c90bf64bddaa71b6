"""Selections on the GPU, looked at one successor at a time: each that is returned is a successor, with the score that it has, in its place; and it is the same whenever it is made."""
import ctypes as C

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
