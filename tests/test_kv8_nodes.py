"""Graph nodes over the paged 8-bit cache (B200_EXT_KV8_STORE, B200_EXT_KV8_ATTN): supports_op says no to a node that its call would refuse, without a GPU."""
import os
import subprocess
from pathlib import Path

import koboldcpp_b200.lib as L

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstdint>
#include <cstring>
#include <functional>
#include "b200_ggml_backend.h"
#include "b200_ggml_ops.h"
#include "b200_kv8.h"

static ggml_tensor tensor(ggml_type type, int64_t ne0, int64_t ne1) {
    ggml_tensor t;
    memset(&t, 0, sizeof(t));
    t.type = type;
    t.ne[0] = ne0; t.ne[1] = ne1; t.ne[2] = t.ne[3] = 1;
    t.nb[0] = 4; t.nb[1] = 4 * (size_t)ne0; t.nb[2] = t.nb[3] = t.nb[1] * (size_t)ne1;
    return t;
}
static void set_f(ggml_tensor &t, int i, float x) { memcpy(&t.op_params[i], &x, 4); }

struct Nodes {  // 2 kv heads of 64 and 48 values, 6 query heads, 5 tokens of 3 sequences
    ggml_tensor k = tensor(GGML_TYPE_F32, 128, 5), v = tensor(GGML_TYPE_F32, 96, 5), info = tensor(GGML_TYPE_I32, 3, 4), table = tensor(GGML_TYPE_I32, 4, 7);
    ggml_tensor pages = tensor(GGML_TYPE_F32, (int64_t)b200_kv8_page_bytes(16, 2, 64, 48) / 4, 9), stored = pages;
    ggml_tensor q = tensor(GGML_TYPE_F32, 384, 5), out = tensor(GGML_TYPE_F32, 288, 5), sink = tensor(GGML_TYPE_F32, 6, 1), ws = tensor(GGML_TYPE_F32, 1, 1);
    Nodes() {
        for (ggml_tensor *t : {&stored, &out}) {
            t->op = GGML_OP_MAP_CUSTOM1;
            t->op_params[0] = (int32_t)B200_EXT_TAG;
            t->op_params[2] = 16; t->op_params[3] = 2; t->op_params[4] = 64; t->op_params[5] = 48;
        }
        stored.op_params[1] = B200_EXT_KV8_STORE;
        out.op_params[1] = B200_EXT_KV8_ATTN;
        set_f(out, 6, 0.125f);
        b200_kv8_attn_args a = {};
        a.cache = {nullptr, 9, 16, 2, 64, 48, 0};
        ws = tensor(GGML_TYPE_F32, (int64_t)(b200_kv8_attn_workspace_bytes(&a) + 3) / 4, 1);
        link();
    }
    void link() {
        ggml_tensor *s[] = {&k, &v, &info, &table, &pages}, *o[] = {&q, &stored, &info, &table, &sink, &ws};
        memcpy(stored.src, s, sizeof(s));
        memcpy(out.src, o, sizeof(o));
    }
};

int main() {
    ggml_backend_reg_t reg = ggml_backend_b200_reg();
    ggml_backend_dev_t dev = reg->iface.get_device(reg, 0);
    int bad = 0;
    auto expect = [&](const char *what, bool store, bool yes, const std::function<void(Nodes &)> &change) {
        Nodes n;
        change(n);
        if (dev->iface.supports_op(dev, store ? &n.stored : &n.out) != yes) { printf("%s: expected %s\n", what, yes ? "yes" : "no"); bad++; }
    };
    expect("store", true, true, [](Nodes &) {});
    expect("attention", false, true, [](Nodes &) {});
    expect("without a sink", false, true, [](Nodes &n) { n.out.src[4] = nullptr; });
    expect("window and cap", false, true, [](Nodes &n) { n.out.op_params[7] = 20; n.out.op_params[8] = 3; set_f(n.out, 9, 30.0f); });
    expect("no tokens", false, true, [](Nodes &n) { n.q.ne[1] = n.out.ne[1] = 0; });
    expect("window below zero", false, false, [](Nodes &n) { n.out.op_params[7] = -1; });
    expect("kept tokens below zero", false, false, [](Nodes &n) { n.out.op_params[8] = -1; });
    expect("cap below zero", false, false, [](Nodes &n) { set_f(n.out, 9, -1.0f); });
    expect("cap that is no number", false, false, [](Nodes &n) { set_f(n.out, 9, NAN); });
    expect("scale that is no number", false, false, [](Nodes &n) { set_f(n.out, 6, NAN); });
    expect("small workspace", false, false, [](Nodes &n) { n.ws.ne[0] -= 4; });
    expect("workspace at an odd place", false, false, [](Nodes &n) { n.ws.data = (void *)4104; });
    expect("rows of q that overlap", false, false, [](Nodes &n) { n.q.nb[1] = 4 * 383; });
    expect("rows of the result that overlap", false, false, [](Nodes &n) { n.out.nb[1] = 4 * 287; });
    expect("a table for more than 2^31 tokens", false, false, [](Nodes &n) { n.table = tensor(GGML_TYPE_I32, (int64_t)1 << 28, 7); });
    expect("too many rows of q", false, false, [](Nodes &n) { n.q = tensor(GGML_TYPE_F32, 384, 400000000); n.out.ne[1] = 400000000; });
    expect("pages at an odd place", false, false, [](Nodes &n) { n.stored.data = (void *)4104; });
    expect("store: rows of k that overlap", true, false, [](Nodes &n) { n.k.nb[1] = 4 * 127; });
    expect("store: rows of v that overlap", true, false, [](Nodes &n) { n.v.nb[1] = 4; });
    expect("store: a table for more than 2^31 tokens", true, false, [](Nodes &n) { n.table = tensor(GGML_TYPE_I32, (int64_t)1 << 28, 7); });
    expect("store: pages at an odd place", true, false, [](Nodes &n) { n.pages.data = (void *)4104; });
    expect("store: other sizes of pages", true, false, [](Nodes &n) { n.stored.op_params[2] = 32; });
    return bad != 0;
}
"""


def test_nodes_that_their_calls_refuse(tmp_path):
    src = tmp_path / "nodes.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "include"), str(src), str(L.LIB_PATH), "-o", str(tmp_path / "nodes"), f"-Wl,-rpath,{Path(L.LIB_PATH).parent}"], check=True)
    r = subprocess.run([str(tmp_path / "nodes")], capture_output=True, text=True, env={**os.environ, "B200_DRY_RUN": "1"})
    assert r.returncode == 0, r.stdout + r.stderr
