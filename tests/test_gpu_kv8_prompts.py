"""Attention over the paged 8-bit cache with enough new tokens for the tensor cores' kernel, on the GPU against tests/kv8_ref.py; bounds as in test_gpu_kv8.py.

Steps of a few thousand query rows over all heads: blocks of 128 rows whose tiles one CTA or several walk, blocks of 256 rows, sequences of few rows among them (the
other kernel's), and workspaces and streams that serve both.
"""
import copy
import ctypes as C
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Kv8AttnArgs, Kv8LoadArgs, Kv8StoreArgs, check, lib
from test_gpu_kv8 import Case, attend, dev, rounded
from test_gpu_kv8 import compare as compare_all

pytestmark = pytest.mark.gpu


def compare(case, q, name, n_head, scale, got, **opt):
    """The first kv heads, one in the middle and the last (the reference takes its time)."""
    group = n_head // case.heads
    kv = sorted({h for h in (0, 1, 2, 3, case.heads // 2, case.heads - 1) if h < case.heads})
    heads = [h * group + i for h in kv for i in range(group)]
    some = copy.copy(case)
    some.pool = copy.copy(case.pool)
    some.heads = some.pool.heads = len(kv)
    some.pool.put(*(x[:, kv] for x in (case.pool.k, case.pool.v, case.pool.ks, case.pool.vs)))
    if opt.get("sink") is not None:
        opt["sink"] = [opt["sink"][h] for h in heads]
    return compare_all(some, q[:, heads], name, len(heads), scale, got[:, heads], **opt)

STEPS = {
    "prompt": [(0, 150)], "behind": [(777, 131)], "far behind": [(2100, 130)], "ragged": [(0, 70), (300, 1), (31, 65), (5, 0), (64, 9), (2, 33), (1500, 40)],
    "many": [(7 * i % 90, 12) for i in range(13)], "mixed": [(1000, 2), (0, 128), (900, 1), (127, 129)],
}
SHAPES = [
    # name, n_head, heads, dim, vdim, page
    ("bf16", 32, 8, 128, 128, 16), ("f32", 32, 2, 64, 64, 32), ("f16", 40, 8, 112, 48, 64), ("f32", 33, 3, 128, 16, 128), ("bf16", 64, 64, 16, 128, 16), ("f32", 48, 1, 80, 96, 16),
    ("f32", 64, 32, 128, 128, 64), ("f16", 34, 17, 64, 32, 16), ("bf16", 36, 6, 32, 64, 128),
]


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("name,n_head,heads,dim,vdim,page", SHAPES)
def test_prompts(step, name, n_head, heads, dim, vdim, page):
    case = Case(STEPS[step], page, heads, dim, vdim, seed=len(step) + dim)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, n_head, dim)), name)
    got, _ = attend(case, cache, q, name, n_head, dim ** -0.5)
    assert compare(case, q, name, n_head, dim ** -0.5, got) == case.tokens
    case.same_pool()


OPTIONS = [dict(window=40), dict(window=40, keep=3), dict(window=1), dict(window=300, keep=200), dict(window=7, keep=100000), dict(window=500, keep=64), dict(sink=True),
           dict(sink=True, window=20, keep=1), dict(softcap=4.0), dict(softcap=30.0, sink=True, window=64), dict(max_new=131), dict(f16=1), dict(f16=1, window=33, keep=5), dict(negative=True)]


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("name,n_head,heads,dim,vdim,page", [("f32", 32, 8, 128, 128, 16), ("bf16", 33, 3, 64, 64, 32), ("f16", 70, 70, 128, 64, 64)])
@pytest.mark.parametrize("step", ["behind", "ragged", "many"])
def test_prompts_options(step, opt, name, n_head, heads, dim, vdim, page):
    case = Case(STEPS[step], page, heads, dim, vdim, seed=21)
    cache = case.upload()
    opt = dict(opt)
    if opt.get("sink"):
        opt["sink"] = np.float32(case.rng.standard_normal(n_head) * 2).tolist()
        opt["sink"][0] = -np.inf  # no sink for this head
    q = rounded(case.rng.standard_normal((case.tokens, n_head, dim)) * 2, name)
    scale = -dim ** -0.5 if opt.pop("negative", False) else dim ** -0.5
    got, _ = attend(case, cache, q, name, n_head, scale, **opt)
    compare(case, q, name, n_head, scale, got, **opt)


@pytest.mark.parametrize("extra,shift", [(1, 0), (0, 1), (8, 8), (5, 3)])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_prompts_of_strided_rows(name, extra, shift):
    case = Case(STEPS["ragged"], 16, 4, 64, 48, seed=22)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, 32, 64)), name)
    got, whole = attend(case, cache, q, name, 32, 0.125, extra=extra, shift=shift)
    compare(case, q, name, 32, 0.125, got)
    plain, _ = attend(case, cache, q, name, 32, 0.125)
    assert (plain == got).all()
    if extra:  # what lies between rows
        between = torch.as_strided(whole, (case.tokens + 2, extra), (32 * 48 + extra, 1), shift + 32 * 48)
        assert torch.equal(between, torch.full_like(between, 3.0))


@pytest.mark.parametrize("n_head,heads", [(32, 4), (80, 80)])
def test_prompts_over_pages_that_are_not_there(n_head, heads):
    """In front of a window, in the middle, all of them: such tokens are not seen, and who sees nothing gets zeros, with a sink or without."""
    case = Case([(700, 60), (40, 33), (0, 70)], 16, heads, 64, 64, seed=23, gone=[(0, 0), (0, 1), (0, 17), (0, 20), (0, 21), (0, 22), (0, 23), (1, 1), (2, 0), (2, 1), (2, 4)])
    case.table[case.order[0], 40] = case.n_pages + 7
    cache = case.upload()
    q = case.rng.standard_normal((case.tokens, n_head, 64)).astype(np.float32).astype(np.float64)
    for opt in (dict(), dict(sink=np.linspace(-2, 2, n_head).tolist()), dict(window=30), dict(window=300, keep=40)):
        got, _ = attend(case, cache, q, "f32", n_head, 0.125, **opt)
        compare(case, q, "f32", n_head, 0.125, got, **opt)
        assert (got[case.first[2]:case.first[2] + 32] == 0).all()


@pytest.mark.parametrize("n_head,heads", [(32, 4), (80, 80)])
def test_prompts_values_that_are_not_finite_reach_only_who_sees_them(n_head, heads):
    case = Case([(0, 70), (1200, 60)], 16, heads, 128, 128, seed=24)
    t = case.table
    case.pool.vs[t[case.order[0], 1], 0] = np.nan   # its first 16 tokens do not see this page
    case.pool.ks[t[case.order[0], 2], 1] = np.nan
    case.pool.ks[t[case.order[1], 30], 2] = np.nan  # in one of several stretches
    case.pool.vs[t[case.order[1], 70], 3] = np.nan
    cache = case.upload()
    q = case.rng.standard_normal((case.tokens, n_head, 128)).astype(np.float32).astype(np.float64)
    for opt in (dict(), dict(window=200), dict(f16=1), dict(sink=[0.25] * n_head)):
        got, _ = attend(case, cache, q, "f32", n_head, 0.088, **opt)
        compare(case, q, "f32", n_head, 0.088, got, **opt)
        assert np.isnan(got).any() and np.isfinite(got[:16]).all()
    # a query that is not finite: its own head and token
    for s in (case.pool.ks, case.pool.vs):
        s[np.isnan(s)] = 0.01
    cache = case.upload()
    q[4, 6, 9] = np.nan
    q[case.first[1] + 9, 3, 5] = np.inf
    got, _ = attend(case, cache, q, "f32", n_head, 0.088)
    want = np.zeros(got.shape[:2], bool)
    want[4, 6] = want[case.first[1] + 9, 3] = True
    assert (np.isnan(got) == want[:, :, None]).all()


def test_prompts_rows_and_scales_far_from_one():
    """Rows of q of all magnitudes, scales of keys and values that differ by powers of ten between pages and heads, and pages of zeros."""
    case = Case([(900, 64), (70, 70)], 16, 4, 128, 128, seed=25)
    rng = case.rng
    case.pool.ks[:] = np.float32(0.02) * (10.0 ** rng.integers(-3, 1, case.pool.ks.shape))
    case.pool.vs[:] = np.float32(0.02) * (10.0 ** rng.integers(-6, 7, case.pool.vs.shape))
    case.pool.vs[case.table[case.order[0], 3]] = 0
    case.pool.ks[case.table[case.order[0], 5]] = 0
    cache = case.upload()
    q = rng.standard_normal((case.tokens, 32, 128)) * 10.0 ** (np.arange(32) % 8 - 7)[None, :, None]
    q[1, 2] = 0
    q = q.astype(np.float32).astype(np.float64)
    for factor, scale in ((1.0, 0.088), (1e-30, 0.088 * 1e30), (1e30, 0.088e-30)):
        x = np.float32(q * factor).astype(np.float64)
        got, _ = attend(case, cache, x, "f32", 32, scale)
        compare(case, x, "f32", 32, scale, got)


def test_prompts_the_same_call_gives_the_same_bits():
    case = Case([(2100, 70), (3000, 2), (5, 64)], 16, 4, 128, 128, seed=26)
    cache = case.upload()
    q = case.rng.standard_normal((case.tokens, 32, 128)).astype(np.float32)
    a, _ = attend(case, cache, q, "f32", 32, 0.088)
    for _ in range(3):
        b, _ = attend(case, cache, q, "f32", 32, 0.088)
        assert (a == b).all()


def test_a_workspace_serves_heads_of_all_sizes():
    """Partial results of one call lie where no other call expects zeros, whatever the sizes of heads."""
    one, two, three = Case([(900, 1)] * 40, 16, 4, 128, 128, seed=27), Case([(1000, 1)] * 40, 32, 4, 64, 64, seed=28), Case([(700, 1)] * 20, 16, 4, 256, 256, seed=29)
    four = Case([(1500, 130), (40, 3)], 16, 4, 128, 128, seed=30)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for case, n_head in ((one, 8), (two, 8), (three, 4), (two, 4), (four, 32), (two, 8), (four, 32), (one, 4), (two, 8)):
        cache = case.upload()
        q = case.rng.standard_normal((case.tokens, n_head, case.dim)).astype(np.float32).astype(np.float64)
        got, _ = attend(case, cache, q, "f32", n_head, 0.1, ws=ws)
        compare(case, q, "f32", n_head, 0.1, got)


def test_two_streams_with_a_workspace_each():
    cases = [Case([(1500, 130), (40, 3)], 16, 4, 128, 128, seed=31), Case([(2000, 4), (100, 90)], 32, 8, 64, 64, seed=32)]
    streams = [torch.cuda.Stream() for _ in cases]
    calls, kept = [], []
    for case, stream in zip(cases, streams):
        cache = case.upload()
        q = case.rng.standard_normal((case.tokens, 64, case.dim)).astype(np.float32)
        tq, out = dev(q), torch.zeros(case.tokens, 64 * case.vdim, device="cuda")
        a = Kv8AttnArgs(cache, tq.data_ptr(), 64 * case.dim, out.data_ptr(), 64 * case.vdim, *case.where(), case.tokens, 0, 64, L.F32, None, 0, 0, 0.1, 0.0, 0)
        ws = torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
        calls.append((a, ws, stream))
        kept.append((q, tq, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for a, ws, stream in calls:
            check(lib().b200_op_kv8_attn(C.byref(a), ws.data_ptr(), ws.numel(), stream.cuda_stream))
    torch.cuda.synchronize()
    for case, (q, _, out) in zip(cases, kept):
        got = out.double().cpu().numpy().reshape(case.tokens, 64, case.vdim)
        compare(case, q.astype(np.float64), "f32", 64, 0.1, got)


@pytest.mark.parametrize("n_head,heads", [(32, 4), (80, 80)])
def test_captured_prompts(n_head, heads):
    """Lengths and places may change between replays of a graph, up to the tokens that it was captured with."""
    case = Case([(1100, 70), (900, 60)], 16, heads, 64, 64, seed=33)
    cache = case.upload()
    q = case.rng.standard_normal((130, n_head, 64)).astype(np.float32).astype(np.float64)
    tq, out = dev(q.astype(np.float32)), torch.zeros(130, n_head * 64, device="cuda")
    a = Kv8AttnArgs(cache, tq.data_ptr(), n_head * 64, out.data_ptr(), n_head * 64, *case.where(), 130, 0, n_head, L.F32, None, 0, 0, 0.125, 0.0, 0)
    ws = torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
    stream, graph = C.c_void_p(), C.c_void_p()
    check(lib().b200_stream_create(C.byref(stream)))
    torch.cuda.synchronize()
    check(lib().b200_graph_begin_capture(stream))
    check(lib().b200_op_kv8_attn(C.byref(a), ws.data_ptr(), ws.numel(), stream))
    check(lib().b200_graph_end_capture(stream, C.byref(graph)))
    for seqs in ([(1100, 70), (900, 60)], [(0, 128), (7, 2)], [(1169, 1), (0, 129)], [(200, 3), (300, 5)], [(1000, 0), (830, 130)]):
        case.seqs, case.new = seqs, [m for _, m in seqs]
        case.first = [0, seqs[0][1]]
        case.d_info.copy_(case.info())
        out.fill_(3.0)
        torch.cuda.synchronize()
        check(lib().b200_graph_launch(graph, stream))
        check(lib().b200_stream_synchronize(stream))
        got = out.double().cpu().numpy().reshape(130, n_head, 64)
        assert compare(case, q, "f32", n_head, 0.125, got) == sum(case.new)
        assert (got[sum(case.new):] == 3.0).all()
    check(lib().b200_graph_destroy(graph))
    check(lib().b200_stream_destroy(stream))


def test_prompts_of_as_many_sequences_as_a_step_may_have():
    case = Case([(i % 40, 9 if i % 8 == 0 else 1) for i in range(1024)], 16, 1, 64, 64, seed=34)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, 8, 64)), "bf16")
    got, _ = attend(case, cache, q, "bf16", 8, 0.125)
    assert compare(case, q, "bf16", 8, 0.125, got) == case.tokens


@pytest.mark.parametrize("n_head,heads,name", [(64, 4, "f32"), (80, 80, "bf16"), (8, 2, "f32")])
def test_steps_that_say_what_cannot_be(n_head, heads, name):
    """Numbers of a step at the ends of 32 bits: such sequences have nothing in the step, and the others get what is theirs (but where the first tokens no longer ascend)."""
    case = Case([(300, 30), (0, 0), (40, 40), (77, 9)], 16, heads, 64, 64, seed=35)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, n_head, 64)), name)
    least, most, f = -2 ** 31, 2 ** 31 - 1, case.first[2]
    fine = copy.copy(case)
    fine.seqs, fine.new = [(300, 30), (0, 0), (40, 0), (77, 9)], [30, 0, 0, 9]
    for column, value in ((0, least), (0, most), (1, least), (2, least), (2, most), (3, least), (3, most)):
        info = case.info().cpu().numpy()
        info[column, 2] = value
        case.d_info = dev(info)
        got, _ = attend(case, cache, q, name, n_head, 0.125)
        assert (got[f:f + 40] == 3.0).all()
        if column != 0:
            compare(fine, q, name, n_head, 0.125, got)
        k, out = torch.ones(case.tokens, heads * 64, device="cuda"), torch.full((case.tokens, heads * 64), 7.0, device="cuda")
        a = Kv8StoreArgs(cache, k.data_ptr(), heads * 64, k.data_ptr(), heads * 64, *case.where(), case.tokens, L.F32)
        check(lib().b200_op_kv8_store(C.byref(a), None))
        a = Kv8LoadArgs(cache, out.data_ptr(), heads * 64, None, 0, *case.where(), case.tokens, L.F32)
        check(lib().b200_op_kv8_load(C.byref(a), None))
        assert (out[f:f + 40] == 7.0).all()
        if column != 0:
            others = torch.cat([out[:f], out[f + 40:]])
            assert (others - 1).abs().max() <= 0.51 * case.pool.ks.max()
        pages = case.table[case.order[2]]
        pages = pages[pages >= 0]
        assert (case.d_pool.cpu().numpy()[pages] == case.pool.records()[pages]).all()
        case.d_pool.copy_(dev(case.pool.records()))
    # positions behind the table's last entry: as many tokens as 31 bits have room for, which see nothing through a window
    info = case.info().cpu().numpy()
    info[3, 2] = most - 20
    case.d_info = dev(info)
    got, _ = attend(case, cache, q, name, n_head, 0.125, window=100)
    assert (got[f:f + 20] == 0).all() and (got[f + 20:f + 40] == 3.0).all()
    fine.pool = case.pool
    compare(fine, q, name, n_head, 0.125, got, window=100)


@pytest.mark.parametrize("extra", [0, 1])
@pytest.mark.parametrize("n_head,heads,new", [(40, 40, 520), (64, 4, 64)])
def test_sums_of_many_keys_do_not_drift(n_head, heads, new, extra):
    """Means of 12,000 values of one sign (q = 0: every weight is 1).  Between two folds there are 128 additions, each off by less than 2^-23 of a sum that grows evenly: 2^-17 of the
    result, less what the factor gives back.  The sum of the weights takes one rounding for each 64 keys, folding one for each 1024: below 200 2^-24.  Weights: 2^-22."""
    case = Case([(12000, new)], 64, heads, 16, 64, seed=37)
    case.pool.put(case.pool.k, np.abs(case.pool.v.astype(np.int16)), case.pool.ks, case.pool.vs)
    cache = case.upload()
    got, _ = attend(case, cache, np.zeros((new, n_head, 16)), "f32", n_head, 0.25, extra=extra)
    v = case.pool.rows(case.table[case.order[0]], 12000 + new, "v")[0]
    n = np.arange(12001, 12001 + new)
    want = np.repeat((np.cumsum(v, axis=0)[12000:] / n[:, None, None]), n_head // heads, axis=1)
    assert (np.abs(got - want) <= (2.0 ** -17 + 200 * 2.0 ** -24 + 2.0 ** -22) * want).all()


GIVE_UP = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import ctypes as C
import numpy as np
import torch
import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Kv8AttnArgs, check, lib
from test_gpu_kv8_prompts import Case, compare, dev, rounded
seqs, n_head, heads, name = {case!r}
case = Case(seqs, 16, heads, 128, 128, seed=36)
cache = case.upload()
q = rounded(case.rng.standard_normal((case.tokens, n_head, 128)), name)
tq = dev(q.astype(np.float32))
tq = tq if name == "f32" else tq.bfloat16()
out = torch.empty(case.tokens, n_head * 128, dtype=tq.dtype, device="cuda")
a = Kv8AttnArgs(cache, tq.data_ptr(), n_head * 128, out.data_ptr(), n_head * 128, *case.where(), case.tokens, 0, n_head, L.F32 if name == "f32" else L.BF16, None, 0, 0, 0.1, 0.0, 0)
ws = torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
def run(limit):
    out.fill_(float("nan"))
    check(lib().b200_op_kv8_attn_wait(C.byref(a), ws.data_ptr(), ws.numel(), limit, None))
    torch.cuda.synchronize()
    return out.double().cpu().numpy().reshape(case.tokens, n_head, 128)
whole = run(4_000_000_000)
compare(case, q, name, n_head, 0.1, whole)
assert lib().b200_gemm_status() == 0
for limit in (100_000, 20_000, 6_000, 2_000, 700, 200, 0):
    got = run(limit)
    stored = ~np.isnan(got)
    print(limit, stored.mean())
    assert np.array_equal(got[stored], whole[stored]), limit
assert not stored.all() and lib().b200_gemm_status() == 1
assert np.array_equal(run(4_000_000_000), whole)
"""


@pytest.mark.parametrize("case", [([(600, 130), (40, 2)], 32, 4, "f32"), ([(600, 130)], 96, 96, "bf16"), ([(100, 130)], 96, 96, "f32"), ([(3000, 130)], 32, 2, "bf16")])
def test_prompts_whose_waits_run_out(case):
    """In a process of its own: that a kernel gave up is remembered for the life of a process."""
    tests = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", GIVE_UP.format(root=str(tests.parent), tests=str(tests), case=case)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
