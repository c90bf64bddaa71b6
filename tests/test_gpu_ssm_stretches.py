"""Scans in stretches on the GPU against tests/state_stretches.py, whose tolerances say what joining stretches may add."""
import ctypes as C

import numpy as np
import pytest

import state_stretches as S
from koboldcpp_b200.lib import lib
from test_gpu_ssm import Scan, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("begin", ["walked", "still"])
def test_sums_of_d_over_long_stretches(begin):
    """32 stretches of 3968 rows and one of a row, states that only fade: an f32 sum of d would be off by a hundred roundings.  The first stretch is walked from the state, not carried: its rows add
    their own errors, 3968 times that of an exponential (6 u) and of a product (2 u), which is more than all joins together.  Where its d is 0, and its factors 1 exactly, the joins are left."""
    rows, ch, n, stretch = 32 * 3968 + 1, 8, 4, 3968
    s = Scan([(rows, 0, False)], ch, n, "f32", softplus=False, bias=False, gate=False, skip=False)
    d, s.a = S.fading(stretch, ch, n, 2.0, seed=1)
    s.dt[:], s.x[:], s.state[:] = d, 0.0, 1.0
    if begin == "still":
        s.dt[:stretch] = 0.0
    a = s.upload()
    assert lib().b200_ssm_scan_workspace_bytes(C.byref(a)) == 4 * ch * (2 * n + 1) * 33
    run(a)
    h, e, turn = np.ones((ch, n)), np.zeros((ch, n)), stretch * d[:, None] * s.a
    none = np.zeros(ch)
    for t in range(stretch if begin == "walked" else 0):
        h, e = S.step(h, e, d, none, none, np.zeros(n), s.a)
    for _ in range(31):
        e = e * np.exp(turn) + S.carry_error(h, turn)
        h = h * np.exp(turn)
    h, e = S.step(h, e, d, none, none, np.zeros(n), s.a)
    got = s.d_state.get().reshape(s.state.shape)[0]
    assert (np.abs(got - h) <= e).all(), (np.abs(got - h) / e).max()


@pytest.mark.parametrize("rows", [129, 640, 3000])
@pytest.mark.parametrize("n", [4, 16, 33])
@pytest.mark.parametrize("softplus", [True, False])
def test_rows_and_states(rows, n, softplus):
    s = Scan([(rows, 1, False)], 40, n, "f32", softplus=softplus, bias=False, gate=False, skip=False, seed=n + rows)
    s.a = -np.random.default_rng(n).uniform(0.05, 0.2, s.a.shape).astype(np.float32).astype(np.float64)
    if not softplus:
        s.dt *= 0.25
        s.dt = s.dt.astype(np.float32).astype(np.float64)
    a = s.upload()
    size = lib().b200_ssm_scan_workspace_bytes(C.byref(a))
    run(a)
    y, h, tol, e = S.scan(s.x, s.dt, s.b, s.c, s.a, s.state[1], S.stretch_of(size, rows, 40, n), is_softplus=softplus)
    got, state = s.d["dst"].get(), s.d_state.get().reshape(s.state.shape)[1]
    assert (np.abs(got - y) <= tol).all(), (np.abs(got - y) / tol).max()
    assert (np.abs(state - h) <= e).all(), (np.abs(state - h) / e).max()
