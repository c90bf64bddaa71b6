"""Prompts of 16 bits behind so many keys that their sums are folded (more than 4096 with f16 rows, 8192 with bf16), where each block of rows is one CTA's: against tests/kv8_ref.py with the bounds
of test_gpu_kv8.py, which hold for sums of any length once they are folded (2^-15 of the mass leaves room for 512 additions of 2^-24)."""
import ctypes as C

import numpy as np
import pytest
import torch

from koboldcpp_b200.lib import BF16, F16, Kv8AttnArgs, check, lib
from test_gpu_kv8 import Case, attend, dev, rounded
from test_gpu_kv8_prompts import compare

pytestmark = pytest.mark.gpu

OPTIONS = [dict(), dict(window=8800, keep=70), dict(window=300, keep=40), dict(sink=True), dict(gone=True), dict(softcap=20.0)]


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("name,n_head,heads,dim,vdim,page,seqs", [("f16", 80, 80, 64, 48, 64, [(9300, 70), (5, 66)]), ("bf16", 80, 80, 16, 112, 128, [(9300, 70), (8100, 66)]), ("f16", 80, 40, 80, 96, 16, [(9001, 70)])])
def test_folded_rows(name, n_head, heads, dim, vdim, page, seqs, opt):
    opt = dict(opt)
    gone = [(0, e) for e in range(3, 9000 // page, 2)] if opt.pop("gone", False) else []
    case = Case(seqs, page, heads, dim, vdim, seed=vdim, gone=gone)
    cache = case.upload()
    if opt.get("sink"):
        opt["sink"] = np.float32(case.rng.standard_normal(n_head) * 2).tolist()
    q = rounded(case.rng.standard_normal((case.tokens, n_head, dim)) * 1.5, name)
    ws = torch.zeros(160 << 20, dtype=torch.uint8, device="cuda")
    first, _ = attend(case, cache, q, name, n_head, dim ** -0.5, ws=ws, **opt)
    compare(case, q, name, n_head, dim ** -0.5, first, **opt)
    for extra, shift in ((0, 0), (1, 0), (5, 3)):  # once more with the same workspace, and rows at any place
        got, whole = attend(case, cache, q, name, n_head, dim ** -0.5, ws=ws, extra=extra, shift=shift, **opt)
        assert (got == first).all()
        if extra:
            between = torch.as_strided(whole, (case.tokens + 2, extra), (n_head * vdim + extra, 1), shift + n_head * vdim)
            assert torch.equal(between, torch.full_like(between, 3.0))


def test_more_blocks_than_places():
    """Blocks of several waves take the places one after another."""
    case = Case([(4500, 700)], 64, 80, 16, 16, seed=9)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, 80, 16)), "f16")
    ws = torch.zeros(160 << 20, dtype=torch.uint8, device="cuda")
    first, _ = attend(case, cache, q, "f16", 80, 0.25, ws=ws)
    compare(case, q, "f16", 80, 0.25, first)
    again, _ = attend(case, cache, q, "f16", 80, 0.25, ws=ws)
    assert (first == again).all()
    assert int(ws[:4 * 148 * 4].sum()) == 0  # none is taken between calls


def call_of(case, q, n_head, name):
    """An attention call with memory of its own: (arguments, workspace, result, what has to live)."""
    dtype = torch.float16 if name == "f16" else torch.bfloat16
    tq, out = dev(q.reshape(case.tokens, -1).astype(np.float32)).to(dtype), torch.zeros(case.tokens, n_head * case.vdim, dtype=dtype, device="cuda")
    a = Kv8AttnArgs(case.upload(), tq.data_ptr(), n_head * case.dim, out.data_ptr(), n_head * case.vdim, *case.where(), case.tokens, 0, n_head, F16 if name == "f16" else BF16, None, 0, 0, 0.2, 0.0, 0)
    return a, torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda"), out, tq


def test_captured_and_replayed():
    """Lengths change between replays: sums that are folded and sums that are not."""
    case = Case([(9300, 70)], 64, 80, 32, 48, seed=40)
    q = rounded(case.rng.standard_normal((70, 80, 32)), "f16")
    a, ws, out, _kept = call_of(case, q, 80, "f16")
    stream, graph = C.c_void_p(), C.c_void_p()
    check(lib().b200_stream_create(C.byref(stream)))
    torch.cuda.synchronize()
    check(lib().b200_graph_begin_capture(stream))
    check(lib().b200_op_kv8_attn(C.byref(a), ws.data_ptr(), ws.numel(), stream))
    check(lib().b200_graph_end_capture(stream, C.byref(graph)))
    for seqs in ([(9300, 70)], [(100, 70)], [(5000, 41)], [(9300, 70)]):
        case.seqs, case.new = seqs, [seqs[0][1]]
        case.d_info.copy_(case.info())
        out.fill_(3.0)
        torch.cuda.synchronize()
        check(lib().b200_graph_launch(graph, stream))
        check(lib().b200_stream_synchronize(stream))
        got = out.double().cpu().numpy().reshape(70, 80, 48)
        assert compare(case, q, "f16", 80, 0.2, got) == seqs[0][1] and (got[seqs[0][1]:] == 3.0).all()
    check(lib().b200_graph_destroy(graph))
    check(lib().b200_stream_destroy(stream))


def test_two_streams():
    """Two calls at a time, a workspace each."""
    cases = [Case([(9300, 70)], 64, 80, 32, 48, seed=41), Case([(8500, 70)], 128, 80, 16, 64, seed=42)]
    names, streams = ("f16", "bf16"), [torch.cuda.Stream() for _ in range(2)]
    qs = [rounded(case.rng.standard_normal((70, 80, case.dim)), name) for case, name in zip(cases, names)]
    calls = [call_of(case, q, 80, name) for case, q, name in zip(cases, qs, names)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (a, ws, _out, _kept), stream in zip(calls, streams):
            check(lib().b200_op_kv8_attn(C.byref(a), ws.data_ptr(), ws.numel(), stream.cuda_stream))
    torch.cuda.synchronize()
    for case, q, name, call in zip(cases, qs, names, calls):
        compare(case, q, name, 80, 0.2, call[2].double().cpu().numpy().reshape(70, 80, case.vdim))
