"""Graph nodes of a state space layer on the GPU: CONCAT, SSM_CONV and SSM_SCAN by themselves and as a graph that the backend computes, captures and replays, against tests/state_ref.py."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import koboldcpp_b200.lib as L
import state_ref as R
from koboldcpp_b200.lib import Tensor, check, lib

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent


def f32(rng, *shape, std=1.0):
    return (rng.normal(size=shape) * std).astype(np.float32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def tensor(t, ne, strides=None):
    """ggml order: ne[0] is innermost; strides in floats."""
    d = Tensor.contiguous(t.data_ptr(), L.F32, ne)
    for i, s in enumerate(strides or []):
        d.nb[i] = 4 * s
    return C.byref(d)


def near(got, want, tol):
    off = np.abs(got - want) > tol
    assert not off.any(), (int(off.sum()), np.argwhere(off)[:4].tolist())


@pytest.mark.parametrize("taps,channels,rows,seqs", [(1, 5, 3, 2), (4, 64, 1, 3), (4, 70, 65, 2), (3, 33, 200, 1), (16, 40, 130, 2)])
def test_convolution(taps, channels, rows, seqs):
    rng = np.random.default_rng(taps)
    gap = 3
    sx, w = f32(rng, seqs, channels, rows + taps - 1 + gap), f32(rng, channels, taps)
    d_sx, d_w, out = dev(sx), dev(w), torch.full((seqs, rows, channels), 7.0, device="cuda")
    n = rows + taps - 1 + gap
    check(lib().b200_op_ssm_conv_nodes(tensor(d_sx, (rows + taps - 1, channels, seqs), (1, n, n * channels, n * channels * seqs)), tensor(d_w, (taps, channels)), tensor(out, (channels, rows, seqs)), None))
    win = np.stack([sx[:, :, j:j + rows] for j in range(taps)], -1).astype(np.float64) * w[:, None]
    want = win.sum(-1).transpose(0, 2, 1)
    near(out.cpu().numpy(), want, taps * 2.0 ** -24 * np.abs(win).sum(-1).transpose(0, 2, 1))


@pytest.mark.parametrize("n,channels,rows,seqs", [(16, 64, 1, 3), (16, 40, 30, 2), (16, 64, 500, 1), (7, 33, 300, 2), (128, 24, 20, 2)])
def test_scan(n, channels, rows, seqs):
    rng = np.random.default_rng(n + rows)
    x, dt, bc = f32(rng, seqs * rows, channels), f32(rng, seqs * rows, channels), f32(rng, seqs * rows, 2 * n + 5)
    a, s = -np.exp(f32(rng, channels, n) - 2), f32(rng, seqs, channels, n)
    d = [dev(v) for v in (s, x, dt, a, bc)]
    ny = x.size
    out = torch.full((ny + s.size + 8,), 7.0, device="cuda")
    w = bc.shape[1]
    view = lambda off: tensor(d[4].view(-1)[off:], (n, rows, seqs), (1, w, w * rows, w * rows * seqs))  # noqa: E731
    args = [tensor(d[0], (n, channels, seqs)), tensor(d[1], (channels, rows, seqs)), tensor(d[2], (channels, rows, seqs)), tensor(d[3], (n, channels)), view(0), view(n), tensor(out, (ny + s.size,))]
    need = lib().b200_op_ssm_scan_nodes_workspace_bytes(args[0], args[1])
    ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")
    check(lib().b200_op_ssm_scan_nodes(*args, ws.data_ptr(), need, None))
    info = np.array([np.arange(seqs) * rows, [rows] * seqs, np.arange(seqs), [0] * seqs])
    f = lambda v: v.astype(np.float64)  # noqa: E731
    y, state, tol, st_tol = R.scan(f(x), f(dt), f(bc[:, :n]), f(bc[:, n:2 * n]), None, f(a), None, None, info, f(s), True, np.zeros((seqs * rows, channels)), "f32")
    got = out.cpu().numpy()
    near(got[:ny].reshape(y.shape), y, tol)
    near(got[ny:ny + s.size].reshape(state.shape), state, st_tol)
    assert (got[ny + s.size:] == 7).all() and np.array_equal(d[0].cpu().numpy(), s)


@pytest.mark.parametrize("dim", [0, 1, 2, 3])
def test_concatenation(dim):
    rng = np.random.default_rng(dim)
    ne = [5, 4, 3, 2]
    nb = list(ne)
    nb[dim] = 7
    a, b = f32(rng, *ne[::-1]), f32(rng, *nb[::-1])
    turned = dev(np.ascontiguousarray(b.swapaxes(2, 3)))  # b as it lies when its first two dimensions are turned over
    out = torch.zeros(*[x + y if i == 3 - dim else x for i, (x, y) in enumerate(zip(a.shape, b.shape))], device="cuda")
    d_a = dev(a)
    total = [ne[i] + (nb[i] if i == dim else 0) for i in range(4)]
    check(lib().b200_op_concat(tensor(d_a, ne), tensor(turned, nb, (nb[1], 1, nb[0] * nb[1], nb[0] * nb[1] * nb[2])), tensor(out, total), dim, None))
    assert np.array_equal(out.cpu().numpy(), np.concatenate([a, b], axis=3 - dim))


PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
#include "b200_ggml_backend.h"

static ggml_tensor shape(int64_t ne0, int64_t ne1 = 1, int64_t ne2 = 1) {
    ggml_tensor t;
    memset(&t, 0, sizeof(t));
    t.type = GGML_TYPE_F32;
    t.ne[0] = ne0; t.ne[1] = ne1; t.ne[2] = ne2; t.ne[3] = 1;
    t.nb[0] = 4; t.nb[1] = 4 * (size_t)ne0; t.nb[2] = t.nb[1] * (size_t)ne1; t.nb[3] = t.nb[2] * (size_t)ne2;
    return t;
}
int main(int argc, char **argv) {  // channels states taps rows sequences; inputs from stdin: tail x w dt a b c s; results to stdout, twice
    const int64_t ch = atoi(argv[1]), n = atoi(argv[2]), k = atoi(argv[3]), t = atoi(argv[4]), q = atoi(argv[5]);
    ggml_backend_t be = ggml_backend_b200_init(0);
    ggml_backend_buffer_type_t buft = ggml_backend_b200_buffer_type(0);
    ggml_tensor tail = shape(k - 1, ch, q), x = shape(ch, t, q), w = shape(k, ch), dt = shape(ch, t, q), a = shape(n, ch), b = shape(n, t, q), c = shape(n, t, q), s = shape(n, ch, q);
    const int layers = 4;  // all alike: a graph of so many nodes is captured
    std::vector<ggml_tensor> xt(layers, x), both(layers, shape(k - 1 + t, ch, q)), conv(layers, shape(ch, t, q)), u(layers, shape(ch, t, q)), out(layers, shape(ch * t * q + n * ch * q));
    std::vector<ggml_tensor *> all = {&tail, &x, &w, &dt, &a, &b, &c, &s}, nodes;
    for (int l = 0; l < layers; l++) for (ggml_tensor *i : {&both[l], &conv[l], &u[l], &out[l]}) all.push_back(i);
    size_t total = 0;
    for (ggml_tensor *i : all) total += (i->nb[3] + 255) / 256 * 256;
    ggml_backend_buffer_t buf = buft->iface.alloc_buffer(buft, total);
    char *at = (char *)buf->iface.get_base(buf);
    for (ggml_tensor *i : all) { i->buffer = buf; i->data = at; at += (i->nb[3] + 255) / 256 * 256; }
    for (int i = 0; i < 8; i++) {
        std::vector<char> h(all[i]->nb[3]);
        if (fread(h.data(), 1, h.size(), stdin) != h.size()) return 2;
        buf->iface.set_tensor(buf, all[i], h.data(), 0, h.size());
    }
    for (int l = 0; l < layers; l++) {
        xt[l] = x;  // x turned over, a view as ggml_transpose makes it
        xt[l].ne[0] = x.ne[1]; xt[l].ne[1] = x.ne[0]; xt[l].nb[0] = x.nb[1]; xt[l].nb[1] = x.nb[0];
        xt[l].op = GGML_OP_TRANSPOSE; xt[l].src[0] = &x; xt[l].view_src = &x;
        both[l].op = GGML_OP_CONCAT; both[l].src[0] = &tail; both[l].src[1] = &xt[l];
        conv[l].op = GGML_OP_SSM_CONV; conv[l].src[0] = &both[l]; conv[l].src[1] = &w;
        u[l].op = GGML_OP_UNARY; u[l].op_params[0] = GGML_UNARY_OP_SILU; u[l].src[0] = &conv[l];
        out[l].op = GGML_OP_SSM_SCAN;
        ggml_tensor *src[] = {&s, &u[l], &dt, &a, &b, &c};
        memcpy(out[l].src, src, sizeof(src));
        for (ggml_tensor *i : {&xt[l], &both[l], &conv[l], &u[l], &out[l]}) nodes.push_back(i);
    }
    ggml_cgraph g;
    memset(&g, 0, sizeof(g));
    g.size = g.n_nodes = (int)nodes.size();
    g.nodes = nodes.data();
    for (int run = 0; run < 4; run++) {
        if (be->iface.graph_compute(be, &g) != GGML_STATUS_SUCCESS) return 3;
        be->iface.synchronize(be);
    }
    int64_t launches, replays, captures;
    ggml_backend_b200_get_stats(&launches, &replays, &captures);
    fprintf(stderr, "%lld launches %lld replays %lld captures\n", (long long)launches, (long long)replays, (long long)captures);
    for (ggml_tensor *i : {&u[0], &out[0], &u[layers - 1], &out[layers - 1]}) {
        std::vector<char> h(i->nb[3]);
        buf->iface.get_tensor(buf, i, h.data(), 0, h.size());
        fwrite(h.data(), 1, h.size(), stdout);
    }
    return 0;
}
"""


@pytest.mark.parametrize("channels,n,taps,rows,seqs", [(64, 16, 4, 1, 3), (96, 16, 4, 37, 2), (40, 16, 4, 600, 1)])
def test_a_layer_as_a_graph(tmp_path, channels, n, taps, rows, seqs):
    """A graph as the reference's own builder makes it, computed four times (the later ones from a captured graph): the states come out behind the rows, the inputs stay."""
    rng = np.random.default_rng(rows)
    tail, x, w = f32(rng, seqs, channels, taps - 1), f32(rng, seqs, rows, channels), f32(rng, channels, taps)
    dt, b, c, s = f32(rng, seqs, rows, channels), f32(rng, seqs, rows, n), f32(rng, seqs, rows, n), f32(rng, seqs, channels, n)
    a = -np.exp(f32(rng, channels, n) - 2).astype(np.float32)
    src = tmp_path / "layer.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "include"), str(src), str(L.LIB_PATH), "-o", str(tmp_path / "layer"), f"-Wl,-rpath,{Path(L.LIB_PATH).parent}"], check=True)
    r = subprocess.run([str(tmp_path / "layer"), *map(str, (channels, n, taps, rows, seqs))], input=b"".join(v.tobytes() for v in (tail, x, w, dt, a, b, c, s)), capture_output=True)
    assert r.returncode == 0, r.stderr.decode()
    replays = int(r.stderr.decode().split("launches ")[1].split()[0])
    assert replays >= 1, r.stderr.decode()
    first, got = np.frombuffer(r.stdout, np.float32).reshape(2, -1)
    assert np.array_equal(first, got)
    info = np.array([np.arange(seqs) * rows, [rows] * seqs, np.arange(seqs), [0] * seqs])
    f = lambda v: v.astype(np.float64)  # noqa: E731
    flat = lambda v: f(v).reshape(seqs * rows, -1)  # noqa: E731
    u, _, u_tol = R.conv(flat(x), f(w), None, info, f(tail).transpose(0, 2, 1), True, np.zeros((seqs * rows, channels)), "f32")
    near(got[:u.size].reshape(u.shape), u, u_tol)
    # the scan by the results that the graph had in front of it
    u = f(got[:u.size]).reshape(u.shape)
    y, state, tol, st_tol = R.scan(u, flat(dt), flat(b), flat(c), None, f(a), None, None, info, f(s), True, np.zeros_like(u), "f32")
    near(got[u.size:2 * u.size].reshape(y.shape), y, tol)
    near(got[2 * u.size:].reshape(state.shape), state, st_tol)
