"""include/b200_state.h without a GPU: what the calls refuse, layouts, sizes of workspaces, and the reference that the GPU tests compare with."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import koboldcpp_b200.lib as L
import state_ref as R
from koboldcpp_b200.lib import BeamSelectArgs, SlotState, SsmConvArgs, SsmScanArgs, lib

HEADER = Path(__file__).resolve().parent.parent / "include" / "b200_state.h"
AT = 4096  # an address that is never read: every call below ends before it would be
UNSUPPORTED, INVALID = 1, 2


def test_every_symbol_is_exported_and_bound():
    declared = set(re.findall(r"B200_API\s+[\w\s\*]+?\b(b200_\w+)\s*\(", HEADER.read_text()))
    assert declared == set(L._STATE_SIGS)
    for name in declared:
        assert hasattr(lib(), name)


def test_structures_have_the_header_s_layout(tmp_path):
    import subprocess
    names = {"b200_ssm_conv_args": SsmConvArgs, "b200_ssm_scan_args": SsmScanArgs, "b200_beam_select_args": BeamSelectArgs, "b200_slot_state": SlotState}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "p.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "p")], check=True)
    for line in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, value = line.split()
        c, _, f = name.partition(".")
        assert int(value) == (getattr(names[c], f).offset if f else C.sizeof(names[c])), name


def conv_args(**change):
    f = dict(x=AT, x_stride=8, w=AT, bias=AT, seq_info=AT, tail=AT, slot_stride=24, dst=2 * AT, dst_stride=8, n_seq=1, n_slots=2, n_tokens=3, max_new=0, channels=8, taps=4, silu=1, type=L.F32)
    return SsmConvArgs(**(f | change))


@pytest.mark.parametrize("change,status", [
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(dst=None), INVALID), (dict(tail=None), INVALID), (dict(type=L.Q8_0), UNSUPPORTED), (dict(n_seq=-1), INVALID), (dict(n_seq=65536), INVALID),
    (dict(n_slots=-1), INVALID), (dict(n_tokens=-1), INVALID), (dict(max_new=-1), INVALID), (dict(channels=0), INVALID), (dict(taps=0), INVALID), (dict(taps=17, slot_stride=999), UNSUPPORTED),
    (dict(x_stride=7), INVALID), (dict(dst_stride=7), INVALID), (dict(slot_stride=23), INVALID), (dict(x=AT + 2), INVALID), (dict(dst=AT + 1, type=L.F16), INVALID), (dict(w=AT + 2), INVALID),
    (dict(tail=AT + 1), INVALID), (dict(dst=AT), INVALID), (dict(seq_info=AT + 1), INVALID), (dict(seq_info=None, n_seq=2), INVALID), (dict(seq_info=None, n_seq=3), INVALID),
    (dict(n_tokens=16 * 65535 + 1), UNSUPPORTED)])
def test_convolutions_that_are_refused(change, status):
    assert lib().b200_op_ssm_conv(C.byref(conv_args(**change)), None) == status
    assert lib().b200_last_error()


def scan_args(**change):
    f = dict(x=AT, x_stride=8, dt=AT, dt_stride=8, b=AT, b_stride=32, c=AT, c_stride=32, z=AT, z_stride=8, a=AT, dt_bias=AT, d=AT, seq_info=AT, state=AT, slot_stride=128, dst=2 * AT, dst_stride=8,
             n_seq=1, n_slots=2, n_tokens=3, max_new=0, channels=8, d_state=16, groups=2, softplus=1, type=L.F32)
    return SsmScanArgs(**(f | change))


@pytest.mark.parametrize("change,status", [
    (dict(x=None), INVALID), (dict(dt=None), INVALID), (dict(b=None), INVALID), (dict(c=None), INVALID), (dict(a=None), INVALID), (dict(state=None), INVALID), (dict(dst=None), INVALID),
    (dict(type=L.I32), UNSUPPORTED), (dict(n_seq=-1), INVALID), (dict(n_seq=65536), INVALID), (dict(n_slots=-1), INVALID), (dict(n_tokens=-1), INVALID), (dict(max_new=-1), INVALID),
    (dict(channels=0), INVALID), (dict(d_state=0), INVALID), (dict(groups=0), INVALID), (dict(groups=3), INVALID), (dict(d_state=129, slot_stride=9999, b_stride=999, c_stride=999), UNSUPPORTED),
    (dict(x_stride=7), INVALID), (dict(dt_stride=7), INVALID), (dict(z_stride=7), INVALID), (dict(dst_stride=7), INVALID), (dict(b_stride=31), INVALID), (dict(c_stride=31), INVALID),
    (dict(slot_stride=127), INVALID), ({"from": AT, "from_stride": 127}, INVALID), (dict(x=AT + 2), INVALID), (dict(z=AT + 1, type=L.BF16), INVALID), (dict(a=AT + 2), INVALID), (dict(state=AT + 2), INVALID),
    (dict(dst=AT), INVALID), (dict(seq_info=AT + 2), INVALID), (dict(seq_info=None, n_seq=2), INVALID), (dict(seq_info=None, n_seq=3), INVALID),
    (dict(dst=3 * AT, x=3 * AT, dst_stride=9), INVALID), (dict(dst=3 * AT, dt=3 * AT, dst_stride=9), INVALID), (dict(dst=3 * AT, z=3 * AT, dst_stride=9), INVALID),
    ({"from": AT, "from_stride": 132}, INVALID)])
def test_scans_that_are_refused(change, status):
    assert lib().b200_op_ssm_scan(C.byref(scan_args(**change)), AT, 1 << 30, None) == status
    assert lib().b200_last_error()


def test_a_scan_in_stretches_needs_its_workspace():
    a = scan_args(channels=64, groups=1, slot_stride=1024, x_stride=64, dt_stride=64, z_stride=64, dst_stride=64, n_tokens=4096)
    need = lib().b200_ssm_scan_workspace_bytes(C.byref(a))
    assert need > 0
    for ws, size in ((None, need), (AT, need - 1), (AT + 8, need)):
        assert lib().b200_op_ssm_scan(C.byref(a), ws, size, None) == INVALID
    a.max_new = 1  # one row a sequence: none
    assert lib().b200_ssm_scan_workspace_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("change", [dict(n_seq=0), dict(n_tokens=0), dict(channels=0), dict(d_state=0), dict(groups=0), dict(groups=3), dict(d_state=129)])
def test_no_workspace_for_calls_that_do_nothing(change):
    assert lib().b200_ssm_scan_workspace_bytes(C.byref(scan_args(**change))) == 0
    assert lib().b200_ssm_scan_workspace_bytes(None) == 0


def test_steps_without_rows_or_sequences_do_nothing():
    for change in (dict(n_seq=0), dict(n_tokens=0), dict(n_seq=0, n_tokens=0, seq_info=None)):
        assert lib().b200_op_ssm_conv(C.byref(conv_args(**change)), None) == 0
        assert lib().b200_op_ssm_scan(C.byref(scan_args(**change)), None, 0, None) == 0
    assert lib().b200_op_ssm_conv(None, None) == INVALID and lib().b200_op_ssm_scan(None, None, 0, None) == INVALID


def select_args(**change):
    f = dict(logits=AT, logits_stride=100, score=AT, ended=AT, slot=AT, to_score=2 * AT, to_beam=2 * AT, to_token=2 * AT, to_slot=2 * AT, n_requests=2, n_beams=4, n_vocab=100, n_keep=8, end_token=2,
             type=L.F32)
    return BeamSelectArgs(**(f | change))


@pytest.mark.parametrize("change,status", [
    (dict(logits=None), INVALID), (dict(score=None), INVALID), (dict(to_score=None), INVALID), (dict(to_beam=None), INVALID), (dict(to_token=None), INVALID), (dict(slot=None), INVALID),
    (dict(type=L.Q4_0), UNSUPPORTED), (dict(n_requests=-1), INVALID), (dict(n_beams=0), INVALID), (dict(n_vocab=0), INVALID), (dict(n_keep=0), INVALID), (dict(n_beams=65), UNSUPPORTED),
    (dict(n_keep=129), UNSUPPORTED), (dict(n_requests=16384), UNSUPPORTED), (dict(n_vocab=(1 << 30) + 1, logits_stride=1 << 31), UNSUPPORTED), (dict(logits_stride=99), INVALID), (dict(end_token=100), INVALID), (dict(end_token=-1), INVALID), (dict(logits=AT + 2), INVALID),
    (dict(logits=AT + 1, type=L.F16), INVALID), (dict(score=AT + 2), INVALID), (dict(to_token=AT + 2), INVALID), (dict(to_score=AT), INVALID), (dict(to_slot=AT), INVALID)])
def test_selections_that_are_refused(change, status):
    assert lib().b200_op_beam_select(C.byref(select_args(**change)), AT, 1 << 30, None) == status
    assert lib().b200_last_error()


def test_a_selection_needs_its_workspace():
    a = select_args()
    need = lib().b200_beam_select_workspace_bytes(C.byref(a))
    assert need > 0
    for ws, size in ((None, need), (AT, need - 1), (AT + 4, need)):
        assert lib().b200_op_beam_select(C.byref(a), ws, size, None) == INVALID
    assert lib().b200_op_beam_select(None, AT, 1 << 20, None) == INVALID
    assert lib().b200_beam_select_workspace_bytes(None) == 0
    a.n_requests = 0
    assert lib().b200_op_beam_select(C.byref(a), None, 0, None) == 0


@pytest.mark.parametrize("states,change,status", [
    ([(AT, 64, 64)], dict(n=-1), INVALID), ([(AT, 64, 64)], dict(n_slots=-1), INVALID), ([(AT, 64, 64)], dict(n=1025), UNSUPPORTED), ([(AT, 64, 64)], dict(n_slots=4097), UNSUPPORTED),
    ([(AT, 64, 64)], dict(src=None), INVALID), ([(AT, 64, 64)], dict(dst=None), INVALID), ([(AT, 64, 64)], dict(src=AT + 2), INVALID), ([(AT, 64, 64)], dict(refused=AT + 2), INVALID),
    ([(None, 64, 64)], {}, INVALID), ([(AT, 60, 64)], {}, INVALID), ([(AT, 64, -4)], {}, INVALID), ([(AT, 64, 64), (AT + 2, 64, 64)], {}, INVALID), ([(AT, 66, 64)], {}, INVALID), ([(AT, 64, 62)], {}, INVALID),
    ([(AT, 1 << 62, 1 << 62)], {}, UNSUPPORTED)])
def test_reorderings_that_are_refused(states, change, status):
    f = dict(src=AT, dst=AT, n=3, n_slots=4, refused=None) | change
    s = (SlotState * len(states))(*[SlotState(*x) for x in states])
    assert lib().b200_op_state_reorder(s, len(s), f["src"], f["dst"], f["n"], f["n_slots"], f["refused"], None) == status
    assert lib().b200_last_error()


def test_reorderings_of_nothing():
    assert lib().b200_op_state_reorder(None, 0, None, None, 0, 4, None, None) == 0
    assert lib().b200_op_state_reorder(None, -1, AT, AT, 1, 4, None, None) == INVALID
    assert lib().b200_op_state_reorder(None, 1, AT, AT, 1, 4, None, None) == INVALID


# ------------------------------------------------------------------------------------------------ the reference
def test_the_scan_is_the_sum_over_all_rows_before():
    """h_t = sum_s exp(a sum of d behind s) d_s x_s b_s, written out."""
    rng = np.random.default_rng(0)
    t, ch, n = 6, 4, 3
    x, dt, b, c = (rng.normal(size=s) for s in ((t, ch), (t, ch), (t, n), (t, n)))
    a, state = -rng.uniform(0.5, 2, size=(ch, n)), rng.normal(size=(2, ch, n))
    y, s, _, _ = R.scan(x, dt, b, c, None, a, None, None, [[0], [t], [1], [0]], state, True, np.zeros((t, ch)), "f32")
    d = np.log1p(np.exp(dt))
    for i in range(t):
        h = state[1] * np.exp(a * d[:i + 1].sum(0)[:, None])
        for j in range(i + 1):
            h = h + np.exp(a * d[j + 1:i + 1].sum(0)[:, None]) * (d[j] * x[j])[:, None] * b[j]
        assert np.allclose(y[i], (h * c[i]).sum(1), rtol=1e-12)
    assert np.allclose(s[1], h, rtol=1e-12) and np.array_equal(s[0], state[0])


def test_selections_go_by_score_then_beam_then_token():
    logits = np.array([[0.0, 0.0, -np.inf, 0.0], [np.nan, 1.0, 1.0, 1.0], [5.0] * 4, [np.inf, 1.0, np.inf, 0.0]])
    score, beam, token, slot = R.select(logits, np.array([-1.0, -1.0, -np.inf, -0.5]), None, np.arange(4), 4, 9, 0)
    assert token.tolist() == [[0, 2, 0, 1, 3, 1, 2, 3, -1]] and beam.tolist() == [[3, 3, 0, 0, 0, 1, 1, 1, -1]] and slot.tolist() == beam.tolist()
    assert np.allclose(score[0, :8], [-0.5 - np.log(2)] * 2 + [-1 - np.log(3)] * 6)
