"""More calls of include/b200_state.h that are refused, on the host: results over inputs, sizes that no index of the kernels reaches."""
import ctypes as C

import pytest

from koboldcpp_b200.lib import lib
from test_state_host import AT, INVALID, select_args

HERE = 1 << 20  # results, far from everything else


@pytest.mark.parametrize("to", ["to_score", "to_beam", "to_token", "to_slot"])
@pytest.mark.parametrize("name,words", [("score", 8), ("ended", 8), ("slot", 8)])
@pytest.mark.parametrize("off", [-15, -1, 0, 1, 7])
def test_selections_over_their_inputs(to, name, words, off):
    """2 requests of 4 beams: 8 numbers of each input; 16 of each result.  Any word in common is refused, not only the same beginning."""
    f = dict(logits=1 << 30, score=2 * HERE, ended=3 * HERE, slot=4 * HERE, to_score=5 * HERE, to_beam=6 * HERE, to_token=7 * HERE, to_slot=8 * HERE)
    a = select_args(**(f | {to: f[name] + 4 * off}))
    assert lib().b200_op_beam_select(C.byref(a), AT, 1 << 30, None) == INVALID
    assert b"in place" in lib().b200_last_error()
