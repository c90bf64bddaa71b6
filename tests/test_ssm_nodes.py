"""Graph nodes of a state space layer (CONCAT, SSM_CONV, SSM_SCAN): supports_op says yes to what the reference's graphs have and no to what the calls refuse, without a GPU."""
import ctypes as C
import os
import subprocess
from pathlib import Path

import pytest

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Tensor, lib

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cstdio>
#include <cstdint>
#include <cstring>
#include <functional>
#include "b200_ggml_backend.h"

static ggml_tensor tensor(int64_t ne0, int64_t ne1 = 1, int64_t ne2 = 1) {
    ggml_tensor t;
    memset(&t, 0, sizeof(t));
    t.type = GGML_TYPE_F32;
    t.ne[0] = ne0; t.ne[1] = ne1; t.ne[2] = ne2; t.ne[3] = 1;
    t.nb[0] = 4; t.nb[1] = 4 * (size_t)ne0; t.nb[2] = t.nb[1] * (size_t)ne1; t.nb[3] = t.nb[2] * (size_t)ne2;
    return t;
}

struct Nodes {  // 24 channels, 4 taps, 16 states, 5 rows of 3 sequences; b and c are columns of a wider product
    ggml_tensor tail = tensor(3, 24, 3), x = tensor(5, 24, 3), both = tensor(8, 24, 3), w = tensor(4, 24), conv = tensor(24, 5, 3);
    ggml_tensor s = tensor(16, 24, 3), dt = tensor(24, 5, 3), a = tensor(16, 24), b = tensor(16, 5, 3), c = tensor(16, 5, 3), out = tensor(24 * 15 + 16 * 24 * 3);
    Nodes() {
        x.nb[0] = 4 * 24; x.nb[1] = 4;  // rows of channels, turned over
        for (ggml_tensor *t : {&b, &c}) { t->nb[1] = 4 * 40; t->nb[2] = 4 * 200; t->nb[3] = 4 * 600; }
        both.op = GGML_OP_CONCAT; both.src[0] = &tail; both.src[1] = &x;
        conv.op = GGML_OP_SSM_CONV; conv.src[0] = &both; conv.src[1] = &w;
        out.op = GGML_OP_SSM_SCAN;
        ggml_tensor *src[] = {&s, &conv, &dt, &a, &b, &c};
        memcpy(out.src, src, sizeof(src));
    }
};

int main() {
    ggml_backend_reg_t reg = ggml_backend_b200_reg();
    ggml_backend_dev_t dev = reg->iface.get_device(reg, 0);
    int bad = 0;
    auto expect = [&](const char *what, int node, bool yes, const std::function<void(Nodes &)> &change) {
        Nodes n;
        change(n);
        ggml_tensor *t[] = {&n.both, &n.conv, &n.out};
        if (dev->iface.supports_op(dev, t[node]) != yes) { printf("%s: expected %s\n", what, yes ? "yes" : "no"); bad++; }
    };
    for (int i = 0; i < 3; i++) expect("as a graph has it", i, true, [](Nodes &) {});
    expect("concat: another dimension", 0, false, [](Nodes &n) { n.both.op_params[0] = 1; });
    expect("concat: no such dimension", 0, false, [](Nodes &n) { n.both.op_params[0] = 4; });
    expect("concat: f16", 0, false, [](Nodes &n) { n.x.type = GGML_TYPE_F16; });
    expect("concat: one of them missing", 0, false, [](Nodes &n) { n.both.src[1] = nullptr; });
    expect("conv: one row too few", 1, false, [](Nodes &n) { n.both.ne[0] = 7; });
    expect("conv: 17 taps", 1, false, [](Nodes &n) { n.w = tensor(17, 24); n.both = tensor(21, 24, 3); });
    expect("conv: other channels", 1, false, [](Nodes &n) { n.w = tensor(4, 25); });
    expect("conv: inputs not side by side", 1, false, [](Nodes &n) { n.both.nb[0] = 8; });
    expect("conv: f16 weights", 1, false, [](Nodes &n) { n.w.type = GGML_TYPE_F16; });
    expect("conv: rows apart", 1, true, [](Nodes &n) { n.both.nb[1] = 4 * 11; n.both.nb[2] = 4 * 300; });
    expect("scan: 129 states", 2, false, [](Nodes &n) { n.s = tensor(129, 24, 3); n.a = tensor(129, 24); n.b = tensor(129, 5, 3); n.c = n.b; n.out.ne[0] = 24 * 15 + 129 * 72; });
    expect("scan: states that are no run", 2, false, [](Nodes &n) { n.s.nb[2] += 4; });
    expect("scan: rows of b at two strides", 2, false, [](Nodes &n) { n.b.nb[2] += 4; });
    expect("scan: rows of c that overlap", 2, false, [](Nodes &n) { n.c.nb[1] = 4 * 15; n.c.nb[2] = 4 * 75; });
    expect("scan: a short result", 2, false, [](Nodes &n) { n.out.ne[0]--; });
    expect("scan: other rows of dt", 2, false, [](Nodes &n) { n.dt.ne[1] = 4; });
    expect("scan: no c", 2, false, [](Nodes &n) { n.out.src[5] = nullptr; });
    expect("scan: f16 rows", 2, false, [](Nodes &n) { n.conv.type = GGML_TYPE_F16; });
    return bad != 0;
}
"""


def test_nodes_that_are_taken_and_refused(tmp_path):
    src = tmp_path / "nodes.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "include"), str(src), str(L.LIB_PATH), "-o", str(tmp_path / "nodes"), f"-Wl,-rpath,{Path(L.LIB_PATH).parent}"], check=True)
    r = subprocess.run([str(tmp_path / "nodes")], capture_output=True, text=True, env={**os.environ, "B200_DRY_RUN": "1"})
    assert r.returncode == 0, r.stdout + r.stderr


AT = 4096


@pytest.mark.parametrize("change,status", [(dict(sx=(7, 24, 3)), 1), (dict(c=(17, 24), sx=(21, 24, 3)), 1), (dict(at=None), 2)])
def test_calls_that_are_refused(change, status):
    at = change.get("at", AT)
    t = [Tensor.contiguous(at, L.F32, change.get(k, v)) for k, v in (("sx", (8, 24, 3)), ("c", (4, 24)), ("dst", (24, 5, 3)))]
    assert lib().b200_op_ssm_conv_nodes(*[C.byref(x) for x in t], None) == status


def test_scans_that_are_refused():
    shapes = dict(s=(16, 64, 1), x=(64, 4096), dt=(64, 4096), a=(16, 64), b=(16, 4096), c=(16, 4096), dst=(64 * 4096 + 16 * 64,))
    def made(**change):
        return [C.byref(Tensor.contiguous(AT, L.F32, (shapes | change)[k])) for k in shapes]
    t = made()
    need = lib().b200_op_ssm_scan_nodes_workspace_bytes(t[0], t[1])
    assert need > 0 and lib().b200_op_ssm_scan_nodes_workspace_bytes(None, None) == 0
    assert lib().b200_op_ssm_scan_nodes(*t, AT, need - 1, None) == 2
    assert lib().b200_op_ssm_scan_nodes(*made(dst=(5,)), AT, need, None) == 1
    assert lib().b200_op_ssm_scan_nodes(*made(a=(16, 63)), AT, need, None) == 1


def test_concatenations_that_are_refused():
    f = lambda *ne: C.byref(Tensor.contiguous(AT, L.F32, ne))  # noqa: E731
    assert lib().b200_op_concat(f(3, 4), f(5, 4), f(8, 4), 4, None) == 2
    assert lib().b200_op_concat(f(3, 4), f(5, 4), f(8, 5), 0, None) == 2
    assert lib().b200_op_concat(f(3, 4), f(5, 4), C.byref(Tensor.contiguous(AT, L.F16, (8, 4))), 0, None) == 1
