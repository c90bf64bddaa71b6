"""More calls of include/b200_state.h that are refused, on the host: results over inputs, sizes that no index of the kernels reaches."""
import ctypes as C

import pytest

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import SlotState, Tensor, lib
from test_state_host import AT, INVALID, UNSUPPORTED, conv_args, scan_args, select_args

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


@pytest.mark.parametrize("over", [1, 1 << 29, (1 << 30) - 1])
def test_more_rows_or_channels_than_an_index_reaches(over):
    """2^30 of either: places of rows and channels are counted in 31 bits, a group of rows or a CTA's channels ahead."""
    big = (1 << 30) + over
    for seqs in (dict(seq_info=AT), dict(seq_info=None, n_seq=1)):
        assert lib().b200_op_ssm_scan(C.byref(scan_args(**(seqs | dict(n_tokens=big)))), AT, 1 << 62, None) == UNSUPPORTED
        assert lib().b200_op_ssm_conv(C.byref(conv_args(**(seqs | dict(n_tokens=big, max_new=5)))), None) == UNSUPPORTED
    wide = dict(channels=big, x_stride=big, dst_stride=big, slot_stride=1 << 62)
    assert lib().b200_op_ssm_conv(C.byref(conv_args(**wide, taps=1)), None) == UNSUPPORTED
    assert lib().b200_op_ssm_scan(C.byref(scan_args(**wide, groups=1, dt_stride=big, z_stride=big)), AT, 1 << 62, None) == UNSUPPORTED
    assert lib().b200_ssm_scan_workspace_bytes(C.byref(scan_args(n_tokens=big))) == 0
    assert lib().b200_ssm_scan_workspace_bytes(C.byref(scan_args(channels=big, groups=1))) == 0


def test_nodes_of_more_rows_than_an_index_reaches():
    rows = 1 << 30
    shapes = dict(s=(4, 8, 1), x=(8, rows + 1), dt=(8, rows + 1), a=(4, 8), b=(4, rows + 1), c=(4, rows + 1), dst=(8 * (rows + 1) + 32,))
    t = [C.byref(Tensor.contiguous(AT, L.F32, shapes[k])) for k in shapes]
    assert lib().b200_op_ssm_scan_nodes_workspace_bytes(t[0], t[1]) == 0
    assert lib().b200_op_ssm_scan_nodes(*t, AT, 1 << 62, None) == UNSUPPORTED


@pytest.mark.parametrize("n,width", [(1, 4096), (8, 4096), (9, 2048), (1024, 32)])
def test_slots_of_more_columns_than_a_launch_counts(n, width):
    """CTAs go through the columns in steps of the grid, which is below 2^16."""
    for columns in ((1 << 31) - 100, (1 << 31) - (1 << 16)):
        s = (SlotState * 1)(SlotState(AT, 1 << 62, width * columns))
        assert lib().b200_op_state_reorder(s, 1, AT, AT, n, 4, None, None) == UNSUPPORTED
