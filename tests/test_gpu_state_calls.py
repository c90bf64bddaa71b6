"""Calls of include/b200_state.h that run at the same time, or are captured, in ways that the other tests do not have."""
import ctypes as C

import pytest
import torch

from koboldcpp_b200.lib import SlotState, check, lib

pytestmark = pytest.mark.gpu


def test_reorderings_on_several_streams_raise_one_number():
    """Every call refuses three of its moves; all streams count into the same word."""
    streams = [torch.cuda.Stream() for _ in range(8)]
    states = [torch.arange(4 * 64, dtype=torch.int32, device="cuda").reshape(4, 64) + i for i in range(8)]
    src, dst = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([1, 0, 9, 2, 3], [0, 1, 2, 0, -1]))
    refused = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = [s[[1, 0, 2, 3]].clone() for s in states]
    torch.cuda.synchronize()
    for _ in range(201):
        for s, x in zip(streams, states):
            one = (SlotState * 1)(SlotState(x.data_ptr(), 256, 256))
            check(lib().b200_op_state_reorder(one, 1, src.data_ptr(), dst.data_ptr(), 5, 4, refused.data_ptr(), s.cuda_stream))
    torch.cuda.synchronize()
    assert refused.item() == 3 * 201 * 8
    assert all(torch.equal(x, w) for x, w in zip(states, want))
