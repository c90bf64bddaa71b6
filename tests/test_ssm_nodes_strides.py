"""Graph nodes of a state space layer whose tensors have strides that nothing goes by: one row of one sequence."""
import ctypes as C
import os
import subprocess
from pathlib import Path

import numpy as np
import pytest

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Tensor, lib
from test_ssm_nodes import AT, PROGRAM

ROOT = Path(__file__).resolve().parent.parent
SHAPES = dict(s=(16, 24, 1), x=(24, 1), dt=(24, 1), a=(16, 24), b=(16, 1), c=(16, 1), dst=(24 + 16 * 24,))


def tensors(at, b_stride):
    t = {k: Tensor.contiguous(at, L.F32, SHAPES[k]) for k in SHAPES}
    for k in ("b", "c"):
        t[k].nb[1] = t[k].nb[2] = t[k].nb[3] = b_stride
    return t


@pytest.mark.parametrize("stride", [0, 4, 60, 64, 4096])
def test_supports_op_and_the_call_agree(tmp_path, stride):
    """What is accepted as a node must not be refused as a call, which ends the process.  (The call is kept from the device by an address that is not aligned, which it looks at last.)"""
    program = PROGRAM.replace("return bad != 0;", f"""
    expect("scan: one row", 2, true, [](Nodes &n) {{
        n.s = tensor(16, 24, 1); n.conv = tensor(24, 1, 1); n.dt = tensor(24, 1, 1); n.b = tensor(16, 1, 1); n.out.ne[0] = 24 + 16 * 24;
        n.b.nb[1] = n.b.nb[2] = n.b.nb[3] = {stride}; n.c = n.b;
    }});
    return bad != 0;""")
    (tmp_path / "nodes.cpp").write_text(program)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "include"), str(tmp_path / "nodes.cpp"), str(L.LIB_PATH), "-o", str(tmp_path / "nodes"), f"-Wl,-rpath,{Path(L.LIB_PATH).parent}"], check=True)
    r = subprocess.run([str(tmp_path / "nodes")], capture_output=True, text=True, env={**os.environ, "B200_DRY_RUN": "1"})
    assert r.returncode == 0, r.stdout + r.stderr
    assert lib().b200_op_ssm_scan_nodes(*[C.byref(t) for t in tensors(AT + 2, stride).values()], None, 0, None) == 2
    assert b"aligned" in lib().b200_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [0, 4, 64, 4096])
def test_one_row(stride):
    import torch

    import state_ref as R
    rng = np.random.default_rng(3)
    h = {k: rng.normal(size=SHAPES[k][::-1]).astype(np.float32) for k in SHAPES}
    h["a"] = -np.exp(h["a"])
    d = {k: torch.from_numpy(v).cuda() for k, v in h.items()}
    t = tensors(0, stride)
    for k in t:
        t[k].data = d[k].data_ptr()
    L.check(lib().b200_op_ssm_scan_nodes(*[C.byref(x) for x in t.values()], None, 0, None))
    f = {k: v.astype(np.float64) for k, v in h.items()}
    y, state, tol, st_tol = R.scan(f["x"], f["dt"], f["b"], f["c"], None, f["a"], None, None, np.array([[0], [1], [0], [0]]), f["s"], True, np.zeros((1, 24)), "f32")
    got = d["dst"].cpu().numpy()
    assert (np.abs(got[:24] - y[0]) <= tol[0]).all() and (np.abs(got[24:].reshape(24, 16) - state[0]) <= st_tol[0]).all()
