"""How far single functions of the scan are from their value, seen through the call: one state, a of 0, b, c and x of 1, so that a sequence's one row is d itself."""
import ctypes as C

import numpy as np
import pytest
import torch

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import SsmScanArgs, check, lib

pytestmark = pytest.mark.gpu


def steps_of(raw, rows):
    """softplus(raw) as single rows or, with two rows whose first has d = 0, as a scan of several rows makes it."""
    n = raw.size
    dt = torch.full((rows, n), -200.0, device="cuda")
    dt[-1] = torch.from_numpy(raw).cuda()
    x, y, one = torch.ones(rows, n, device="cuda"), torch.zeros(rows, n, device="cuda"), torch.ones(rows, 1, device="cuda")
    a, state = torch.zeros(n, 1, device="cuda"), torch.zeros(n, 1, device="cuda")
    args = SsmScanArgs(x=x.data_ptr(), x_stride=n, dt=dt.data_ptr(), dt_stride=n, b=one.data_ptr(), b_stride=1, c=one.data_ptr(), c_stride=1, a=a.data_ptr(), state=state.data_ptr(), slot_stride=n,
                       dst=y.data_ptr(), dst_stride=n, n_seq=1, n_slots=1, n_tokens=rows, channels=n, d_state=1, groups=1, softplus=1, type=L.F32)
    check(lib().b200_op_ssm_scan(C.byref(args), None, 0, None))
    return y[-1].double().cpu().numpy()


# An exponential of the special function unit (2^-22) whose argument's rounding is made good but for 2 u; the polynomial 1.8e-7 with its own roundings; the sum with max(x, 0), a product with x and b each: 3 u.
WORST = 2.0 ** -22 + 1.8e-7 + 5 * 2.0 ** -24


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("lo,hi", [(-85, -30), (-30, -12), (-12, -6), (-6, -2), (-2, 2), (2, 20), (20, 85)])
def test_softplus(rows, lo, hi):
    raw = np.random.default_rng(rows).uniform(lo, hi, 1 << 18).astype(np.float32)
    want = np.logaddexp(0, raw.astype(np.float64))
    off = (steps_of(raw, rows) - want) / want
    print(f"\n{lo} .. {hi}: largest {np.abs(off).max():.2e}, root mean square {np.sqrt((off ** 2).mean()):.2e}, mean {off.mean():.1e}")
    assert np.abs(off).max() <= WORST
    assert abs(off.mean()) <= 2.0 ** -24  # (no side that it errs to by more than half a step)
