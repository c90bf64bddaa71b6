"""The paged 8-bit cache on the GPU against tests/kv8_ref.py (include/b200_kv8.h).

What is stored is compared bit by bit, records whole: quotients are rounded exactly, scales are f32 divisions and products.  Results of attention are held
to bounds made of each case's own numbers.  With E the largest error of a score and w that of a weight relative to itself, a result is off by
(2 E + w) sum_j p_j |v_j| at most, to first order (numerator and denominator each take E), plus its own rounding.
  * Scores: q enters as two f16 (what they leave over: 2^-22 of the row's largest value) or one f16 (2^-11 of each, exact for rows of 8 or 11 bits but for values
    2^-24 of the row's largest); the sum of up to 256 products in f32 is off by less than 2^-17 sum |q k| in any order of additions (256 2^-24 = 2^-16 at the
    very worst with roundings of one sign; the sums run in pieces of 16).  E = (2^-16 + q's) scale max_j sum_d |q_d k_d|, and with a soft cap it only shrinks.
    q's error in terms of sum |q k|: one f16: 2^-11.  Two f16: 2^-22 max|q| sum |k| is below 2^-22 16 sum |q k| for normal q and k (max|q| / mean|q| < 8 over 256
    values, and the products are independent): 2^-18.
  * Weights: exponential and its argument 2^-18 (scores below 64), two f16 2^-22 or one 2^-11, sums in f32 of up to 4096 keys: 2^-24 4096 / 16 (a thread adds every
    16th) = 2^-16.  w = 2^-15 or 2^-11 + 2^-15.
  * Weights far below the row's largest: f16 has steps of 2^-24 and no finer ones, so a weight as it enters the second product is off by 2^-25 too, however small it
    is.  It enters as p_j / max p (at least: the sum that divides is 1 or more in this unit) times its scale times 2^6 / 2^power, 2^power being at most twice the
    largest scale that the row has seen: 2^-25 2^-6 2 = 2^-30 of that scale, times an int8 of at most 127, for each key that is seen.  It shows where a key takes all
    the weight and its value is 0.
"""
import ctypes as C

import numpy as np
import pytest
import torch

import kv8_ref as R
import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Kv8AttnArgs, Kv8Cache, Kv8LoadArgs, Kv8Map, Kv8StoreArgs, check, lib

pytestmark = pytest.mark.gpu

TYPES = {"f32": (L.F32, torch.float32), "f16": (L.F16, torch.float16), "bf16": (L.BF16, torch.bfloat16)}


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda") if dtype is None else torch.from_numpy(np.ascontiguousarray(a)).to("cuda").to(dtype)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rounded(a, name):
    """a as the type holds it, in 64 bits."""
    return torch.from_numpy(np.asarray(a, np.float32)).to(TYPES[name][1]).double().numpy()


class Case:
    """Sequences over a pool: (held, new) each, pages in a mixed order, rows in a mixed order."""

    def __init__(self, seqs, page=16, heads=2, dim=64, vdim=64, seed=0, spare=2, gone=()):
        rng = self.rng = np.random.default_rng(seed)
        self.seqs, self.page, self.heads, self.dim, self.vdim = seqs, page, heads, dim, vdim
        need = [-(-(h + m) // page) for h, m in seqs]
        self.n_rows = len(seqs) + 2
        self.n_pages = sum(need) + spare
        self.pool = R.Pool(self.n_pages, page, heads, dim, vdim, seed)
        mixed = rng.permutation(self.n_pages)
        self.order = rng.permutation(self.n_rows)[:len(seqs)].tolist()
        self.table = np.full((self.n_rows, max(need + [1]) + 1), -1, np.int32)
        at = 0
        for r, n in zip(self.order, need):
            self.table[r, :n] = mixed[at:at + n]
            at += n
        for i, e in gone:
            self.table[self.order[i], e] = -1
        self.new = [m for _, m in seqs]
        self.tokens = sum(self.new)
        self.first = np.concatenate([[0], np.cumsum(self.new)])[:-1].tolist()

    def upload(self):
        # (a copy in a larger allocation: records begin on 128 bytes)
        self.d_pool = dev(self.pool.records())
        self.d_table = dev(self.table)
        self.d_info = self.info()
        return Kv8Cache(self.d_pool.data_ptr(), self.n_pages, self.page, self.heads, self.dim, self.vdim)

    def info(self, held=None, new=None):
        held, new = held or [h for h, _ in self.seqs], new or self.new
        first = np.concatenate([[0], np.cumsum(new)])[:-1]
        return dev(np.array([first, new, self.order, held], np.int32))

    def where(self):
        return self.d_info.data_ptr(), self.d_table.data_ptr(), self.table.shape[1], self.n_rows, len(self.seqs)

    def same_pool(self):
        got, want = self.d_pool.cpu().numpy(), self.pool.records()
        bad = np.argwhere(got != want)
        assert bad.size == 0, f"{len(bad)} bytes differ, first page {bad[0][0]} byte {bad[0][1]} (values end at {self.pool.at})"


def buffer(rows, width, dtype, extra=0, shift=0, fill=None):
    """Rows with a stride of width + extra, beginning `shift` values behind an aligned place; and the tensor that holds them."""
    whole = torch.full((rows * (width + extra) + shift + 16,), 0.0 if fill is None else fill, dtype=dtype, device="cuda")
    return torch.as_strided(whole, (rows, width), (width + extra, 1), shift), whole


PATTERNS = {
    "one token": [(0, 1)], "next token": [(5, 1)], "page begins": [(16, 1)], "page ends": [(15, 1)], "across a page": [(13, 9)], "two pages and a bit": [(0, 37)], "long": [(3, 301)],
    "batch": [(0, 1), (7, 1), (33, 1), (255, 1)], "ragged": [(0, 5), (40, 1), (17, 0), (2, 70), (0, 0), (9, 3)], "nothing first": [(4, 0), (1, 2)], "many": [(i, 1 + i % 3) for i in range(70)],
}


# ------------------------------------------------------------------------------------------------ store and load
def run_store(case, cache, k, v, name, stream=None, tokens=None):
    a = Kv8StoreArgs(cache, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), *case.where(), case.tokens if tokens is None else tokens, TYPES[name][0])
    check(lib().b200_op_kv8_store(C.byref(a), stream))


def rows_of(case, name, loud=1.0, extra=0, shift=0):
    rng = case.rng
    k = rounded(rng.standard_normal((case.tokens, case.heads, case.dim)) * np.exp(0.5 * rng.standard_normal((case.tokens, case.heads, 1))) * loud, name)
    v = rounded(rng.standard_normal((case.tokens, case.heads, case.vdim)) * np.exp(0.5 * rng.standard_normal((case.tokens, case.heads, 1))) * loud, name)
    out = []
    for x, size in ((k, case.dim), (v, case.vdim)):
        t, _ = buffer(case.tokens, case.heads * size, TYPES[name][1], extra, shift)
        t.copy_(torch.from_numpy(x.reshape(case.tokens, -1)))
        out.append(t)
    return k, v, out[0], out[1]


def reference_store(case, k, v):
    for (held, m), r, f in zip(case.seqs, case.order, case.first):
        case.pool.store(case.table[r], k[f:f + m], v[f:f + m], held)


@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("name,page,heads,dim,vdim,extra,shift", [("f32", 16, 2, 64, 64, 0, 0), ("bf16", 32, 3, 128, 128, 0, 0), ("f16", 64, 1, 256, 80, 8, 0), ("f32", 128, 2, 96, 16, 3, 1),
                                                                  ("bf16", 16, 5, 16, 256, 1, 3), ("f16", 128, 2, 112, 192, 0, 2)])
def test_store_and_load(pattern, name, page, heads, dim, vdim, extra, shift):
    case = Case(PATTERNS[pattern], page, heads, dim, vdim, seed=len(pattern))
    cache = case.upload()
    k, v, tk, tv = rows_of(case, name, extra=extra, shift=shift)
    run_store(case, cache, tk, tv, name)
    reference_store(case, k, v)
    case.same_pool()
    # and read back from the start of the sequences
    both = [h + m for h, m in case.seqs]
    out = [buffer(sum(both) + 2, heads * size, TYPES[name][1], extra, shift, fill=7.0) for size in (dim, vdim)]
    info = case.info([0] * len(both), both)
    a = Kv8LoadArgs(cache, out[0][0].data_ptr(), out[0][0].stride(0), out[1][0].data_ptr(), out[1][0].stride(0), info.data_ptr(), *case.where()[1:], sum(both) + 2, TYPES[name][0])
    check(lib().b200_op_kv8_load(C.byref(a), None))
    for (t, whole), which, size in zip(out, "kv", (dim, vdim)):
        want, want_whole = buffer(sum(both) + 2, heads * size, TYPES[name][1], extra, shift, fill=7.0)
        values = np.concatenate([case.pool.rows(case.table[r], n, which)[0] for r, n in zip(case.order, both)]).reshape(sum(both), -1)
        want[:sum(both)] = torch.from_numpy(values.astype(np.float32)).to(TYPES[name][1]).cuda()
        assert torch.equal(whole, want_whole)  # rows behind the last sequence and what lies between rows too


def test_load_of_one_half_and_of_pages_that_are_not_there():
    case = Case([(0, 40), (0, 20)], page=16, heads=2, dim=64, vdim=32, gone=[(0, 1)], seed=3)
    cache = case.upload()
    for which, size in (("k", 64), ("v", 32)):
        out = torch.full((60, 2 * size), 5.0, device="cuda")
        ptr = {"k": (out.data_ptr(), out.stride(0), None, 0), "v": (None, 0, out.data_ptr(), out.stride(0))}[which]
        check(lib().b200_op_kv8_load(C.byref(Kv8LoadArgs(cache, *ptr, *case.where(), 60, L.F32)), None))
        want = np.concatenate([case.pool.rows(case.table[r], n, which)[0] for r, n in zip(case.order, (40, 20))]).reshape(60, -1)
        assert (out.cpu().numpy() == want.astype(np.float32)).all() and (want[16:32] == 0).all()


@pytest.mark.parametrize("loud", [1e-41, 1e-38, 1e-30, 1.0, 1e30])
def test_store_of_all_magnitudes(loud):
    case = Case([(0, 20), (9, 30)], seed=5)
    cache = case.upload()
    k, v, tk, tv = rows_of(case, "f32", loud)
    tk[3] = 0
    k[3] = 0
    run_store(case, cache, tk, tv, "f32")
    reference_store(case, k, v)
    case.same_pool()


def test_store_at_the_border_between_two_steps():
    """Values at half steps (ties go to the even one) and one f32 on either side of them, under scales that are no power of two."""
    case = Case([(0, 16)], heads=1, dim=256, vdim=256, seed=6)
    cache = case.upload()
    scale = np.float32(0.0371)
    half = ((np.arange(-127, 127, dtype=np.float64) + 0.5) * np.float64(scale)).astype(np.float32)
    around = np.stack([half, np.nextafter(half, np.float32(np.inf)), np.nextafter(half, -np.float32(np.inf))])
    k = np.zeros((16, 1, 256), np.float32)
    k[:3, 0, :254] = around
    k[:, 0, 255] = np.float32(127 * np.float64(scale))
    assert np.float32(np.float64(k[:, 0, 255].max()) / 127) == scale
    k[4:7, 0, :254] = around[:, ::-1]
    v = k[::-1].copy()
    run_store(case, cache, dev(k.reshape(16, -1)), dev(v.reshape(16, -1)), "f32")
    reference_store(case, k.astype(np.float64), v.astype(np.float64))
    case.same_pool()


def test_a_page_that_fills_token_by_token():
    case = Case([(0, 1)] * 3, heads=2, dim=32, vdim=48, seed=7)
    case.table[:, :] = -1
    for i, r in enumerate(case.order):
        case.table[r, 0] = i
    cache = case.upload()
    growth = [np.ones(16), np.exp(np.linspace(-3, 3, 16)), np.exp(np.sin(np.arange(16.0)))]
    for t in range(16):
        case.seqs = [(t, 1)] * 3
        k, v, tk, tv = rows_of(case, "f32")
        for i in range(3):
            k[i] = np.float32(k[i] * growth[i][t])
            v[i] = np.float32(v[i] * growth[i][t])
        tk.copy_(torch.from_numpy(k.reshape(3, -1)))
        tv.copy_(torch.from_numpy(v.reshape(3, -1)))
        case.d_info = case.info()
        run_store(case, cache, tk, tv, "f32")
        reference_store(case, k, v)
        case.same_pool()


def test_what_is_not_finite_stays_in_its_page_and_head():
    case = Case([(0, 20), (3, 20), (0, 5)], heads=3, seed=8)
    cache = case.upload()
    k, v, tk, tv = rows_of(case, "f32")
    for t, x, val in ((2, k, np.nan), (25, k, np.inf), (18, v, -np.inf), (41, v, np.nan)):
        x[t, 1, 7] = val
    tk.copy_(torch.from_numpy(k.reshape(45, -1)))
    tv.copy_(torch.from_numpy(v.reshape(45, -1)))
    run_store(case, cache, tk, tv, "f32")
    reference_store(case, k, v)

    def same():  # NaN by what it is, whatever its bits
        case.d_pool = case.d_pool.cpu()
        got = case.d_pool.numpy()
        b = case.pool.at[1]
        scales = got[:, b:b + 24].copy().view(np.float32)
        assert (np.isnan(scales) == np.isnan(np.concatenate([case.pool.ks, case.pool.vs], axis=1))).all()
        scales[np.isnan(scales)] = np.nan
        got[:, b:b + 24] = scales.view(np.uint8)
        for s in (case.pool.ks, case.pool.vs):
            s[np.isnan(s)] = np.nan
        case.same_pool()
        case.d_pool = case.d_pool.cuda()
    same()
    assert np.isnan(case.pool.ks).sum() == 2 and np.isnan(case.pool.vs).sum() == 2
    # it stays until the page is begun anew
    cache = Kv8Cache(case.d_pool.data_ptr(), case.n_pages, case.page, case.heads, case.dim, case.vdim)
    for seqs in ([(20, 1), (23, 1), (5, 1)], [(16, 4), (0, 20), (0, 5)]):
        case.seqs, case.new, case.tokens = seqs, [m for _, m in seqs], sum(m for _, m in seqs)
        case.first = np.concatenate([[0], np.cumsum(case.new)])[:-1].tolist()
        case.d_info = case.info()
        k, v, tk, tv = rows_of(case, "f32")
        run_store(case, cache, tk, tv, "f32")
        reference_store(case, k, v)
        same()
        cache = Kv8Cache(case.d_pool.data_ptr(), case.n_pages, case.page, case.heads, case.dim, case.vdim)


def test_store_leaves_out_what_lies_outside():
    """Pages that are not there (-1, beyond the pool), rows beyond the table's, tokens beyond the batch, positions beyond the table's entries."""
    case = Case([(0, 40), (5, 20), (10, 30), (0, 4)], seed=9, gone=[(0, 1)])
    case.table[case.order[1], 0] = case.n_pages
    cache = case.upload()
    k, v, tk, tv = rows_of(case, "f32")
    info = case.info().cpu().numpy()
    info[2, 3] = case.n_rows       # no such row
    info[3, 2] = 16 * case.table.shape[1] - 5  # 30 tokens, 5 of them within the table (whose last entry is -1)
    case.d_info = dev(info)
    run_store(case, cache, tk, tv, "f32", tokens=case.tokens - 10)  # the last tokens of the third sequence and the fourth are outside
    case.pool.store(case.table[case.order[0]], k[:40], v[:40], 0)
    case.pool.store(case.table[case.order[1]], k[40:60], v[40:60], 5)
    case.same_pool()


# ------------------------------------------------------------------------------------------------ attention
def attend(case, cache, q, name, n_head, scale, tokens=None, stream=None, ws=None, extra=0, shift=0, fill=3.0, **opt):
    """Results [tokens][n_head][vdim] in 64 bits, and the whole buffer."""
    n = q.shape[0]
    tq, _ = buffer(n, n_head * case.dim, TYPES[name][1], extra, shift)
    tq.copy_(torch.from_numpy(q.reshape(n, -1)))
    out, whole = buffer(n + 2, n_head * case.vdim, TYPES[name][1], extra, shift, fill=fill)
    sink = opt.get("sink")
    d_sink = None if sink is None else dev(np.asarray(sink, np.float32))
    a = Kv8AttnArgs(cache, tq.data_ptr(), tq.stride(0), out.data_ptr(), out.stride(0), *case.where(), n if tokens is None else tokens, opt.get("max_new", 0), n_head, TYPES[name][0],
                    None if sink is None else d_sink.data_ptr(), opt.get("window", 0), opt.get("keep", 0), scale, opt.get("softcap", 0.0), opt.get("f16", 0))
    need = lib().b200_kv8_attn_workspace_bytes(C.byref(a))
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda") if ws is None else ws
    check(lib().b200_op_kv8_attn(C.byref(a), ws.data_ptr(), ws.numel(), stream))
    torch.cuda.synchronize()
    assert torch.equal(out[n:], torch.full_like(out[n:], fill))  # rows behind the last sequence
    return out[:n].double().cpu().numpy().reshape(n, n_head, case.vdim), whole


def bound(name, mass, size, want, f16):
    one = name != "f32" or f16
    q = 2.0 ** -11 if one else 2.0 ** -18
    e = (2.0 ** -16 + q) * size[:, :, None]
    w = 2.0 ** -15 + (2.0 ** -11 if one else 0.0)
    eps = torch.finfo(TYPES[name][1]).eps / 2
    return (np.expm1(2 * e) + w) * mass * 1.01 + eps * np.abs(want) + 1e-30


def compare(case, q, name, n_head, scale, got, **opt):
    checked = 0
    for (held, m), r, f in zip(case.seqs, case.order, case.first):
        if m == 0:
            continue
        sink = None if opt.get("sink") is None else np.asarray(opt["sink"], np.float32).astype(np.float64)
        want, mass, size = case.pool.attend(case.table[r], q[f:f + m], held, np.float64(np.float32(scale)), opt.get("window", 0), opt.get("keep", 0), sink, opt.get("softcap", 0.0))
        x = got[f:f + m]
        assert (np.isnan(x) == np.isnan(want)).all(), (held, m)
        loud = np.fmax.reduce(case.pool.vs[[p for p in case.table[r] if 0 <= p < case.n_pages]], axis=0, initial=0.0)  # of each kv head
        keys = np.minimum(held + 1 + np.arange(m), opt["window"] + opt.get("keep", 0) if opt.get("window", 0) else held + m)
        least = 2.0 ** -30 * 127 * keys[:, None, None] * np.repeat(loud, n_head // case.heads)[None, :, None]
        off, most = np.abs(x - want), bound(name, mass, size, want, opt.get("f16", 0)) + least
        fine = np.isfinite(want)
        assert (off[fine] <= most[fine]).all(), (held, m, float(np.max(off[fine] / most[fine])), np.argwhere(off > most)[:5].tolist())
        checked += m
    return checked


ATTN = [
    # name, n_head, heads, dim, vdim, page
    ("f32", 8, 2, 128, 128, 16), ("f32", 4, 4, 64, 64, 32), ("bf16", 10, 2, 128, 128, 64), ("f16", 3, 1, 96, 80, 16), ("f32", 9, 1, 256, 256, 16), ("bf16", 2, 1, 192, 64, 128),
    ("f16", 32, 1, 64, 64, 16), ("f32", 6, 2, 16, 112, 128), ("bf16", 16, 2, 32, 48, 32), ("f32", 40, 2, 80, 96, 64), ("f16", 8, 4, 256, 128, 32),
]
STEPS = {
    "first": [(0, 1)], "one": [(37, 1)], "page end": [(15, 1), (31, 1)], "page begin": [(16, 1), (64, 1), (128, 1)], "batch": [(0, 1), (200, 1), (517, 1), (63, 1), (1, 1)],
    "drafts": [(30, 5), (0, 3), (129, 7)], "long": [(2100, 1)], "ragged": [(0, 40), (77, 0), (5, 1), (300, 17), (0, 1)], "prompt": [(0, 150)], "behind": [(140, 65), (3, 130)],
    "many": [(3 * i, 1) for i in range(75)],
}


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("name,n_head,heads,dim,vdim,page", ATTN)
def test_attention(step, name, n_head, heads, dim, vdim, page):
    case = Case(STEPS[step], page, heads, dim, vdim, seed=len(step) + dim)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, n_head, dim)), name)
    scale = dim ** -0.5
    got, _ = attend(case, cache, q, name, n_head, scale)
    assert compare(case, q, name, n_head, scale, got) == case.tokens
    case.same_pool()


OPTIONS = [dict(window=40), dict(window=40, keep=3), dict(window=1), dict(window=300, keep=200), dict(window=7, keep=100000), dict(sink=True), dict(sink=True, window=20, keep=1), dict(softcap=4.0),
           dict(softcap=30.0, sink=True, window=64), dict(max_new=64), dict(f16=1), dict(f16=1, window=33, keep=5)]


@pytest.mark.parametrize("opt", OPTIONS, ids=str)
@pytest.mark.parametrize("name,n_head,heads,dim,vdim,page", [("f32", 8, 2, 128, 128, 16), ("bf16", 4, 1, 64, 64, 32), ("f16", 6, 2, 96, 256, 64)])
@pytest.mark.parametrize("step", ["batch", "ragged", "long", "behind"])
def test_attention_options(step, opt, name, n_head, heads, dim, vdim, page):
    case = Case(STEPS[step], page, heads, dim, vdim, seed=11)
    cache = case.upload()
    opt = dict(opt)
    if opt.get("sink"):
        opt["sink"] = np.float32(case.rng.standard_normal(n_head) * 2).tolist()
        opt["sink"][0] = -np.inf  # no sink for this head
    q = rounded(case.rng.standard_normal((case.tokens, n_head, dim)) * 2, name)
    scale = dim ** -0.5
    got, _ = attend(case, cache, q, name, n_head, scale, **opt)
    compare(case, q, name, n_head, scale, got, **opt)


@pytest.mark.parametrize("extra,shift", [(1, 0), (0, 1), (8, 8), (5, 3)])
@pytest.mark.parametrize("name", TYPES)
def test_attention_of_strided_rows(name, extra, shift):
    case = Case(STEPS["ragged"], 16, 2, 64, 64, seed=12)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, 4, 64)), name)
    got, whole = attend(case, cache, q, name, 4, 0.125, extra=extra, shift=shift)
    compare(case, q, name, 4, 0.125, got)
    plain, _ = attend(case, cache, q, name, 4, 0.125)
    assert (plain == got).all()
    if extra:  # what lies between rows
        between = torch.as_strided(whole, (case.tokens + 2, extra), (256 + extra, 1), shift + 256)
        assert torch.equal(between, torch.full_like(between, 3.0))


def test_attention_over_pages_that_are_not_there():
    """In front of a window, in the middle, all of them: such tokens are not seen, and who sees nothing gets zeros, with a sink or without."""
    case = Case([(100, 2), (40, 1), (20, 3), (0, 30)], 16, 2, 64, 64, seed=13, gone=[(0, 0), (0, 1), (1, 1), (2, 0), (2, 1), (3, 0)])
    case.table[case.order[0], 3] = case.n_pages + 7
    cache = case.upload()
    q = case.rng.standard_normal((case.tokens, 4, 64)).astype(np.float32).astype(np.float64)
    for opt in (dict(), dict(sink=[0.5, -1.0, 2.0, 0.0]), dict(window=30)):
        got, _ = attend(case, cache, q, "f32", 4, 0.125, **opt)
        compare(case, q, "f32", 4, 0.125, got, **opt)
        f = case.first[2]
        assert (got[f:f + 3] == 0).all() and (got[case.first[3]:case.first[3] + 16] == 0).all()


def test_values_that_are_not_finite_reach_only_who_sees_them():
    case = Case([(50, 3), (90, 1), (0, 40)], 16, 2, 128, 128, seed=14)
    t = case.table
    case.pool.ks[t[case.order[0], 1], 0] = np.nan
    case.pool.vs[t[case.order[1], 0], 1] = np.nan
    case.pool.vs[t[case.order[2], 1], 0] = np.nan   # a prompt: its first 16 tokens do not see this page
    case.pool.ks[t[case.order[2], 2], 1] = np.nan
    cache = case.upload()
    q = case.rng.standard_normal((case.tokens, 8, 128)).astype(np.float32).astype(np.float64)
    for opt in (dict(), dict(window=20), dict(f16=1)):
        got, _ = attend(case, cache, q, "f32", 8, 0.088, **opt)
        compare(case, q, "f32", 8, 0.088, got, **opt)
        assert np.isnan(got).any() and np.isfinite(got[case.first[2]:case.first[2] + 16]).all()
    # a query that is not finite: its own head and token
    q[case.first[1], 3, 5] = np.inf
    q[case.first[2] + 4, 6, 9] = np.nan
    got, _ = attend(case, cache, q, "f32", 8, 0.088)
    assert np.isnan(got[case.first[1], 3]).all() and np.isnan(got[case.first[2] + 4, 6]).all()
    assert np.isfinite(got[case.first[2] + 4, [0, 1, 2, 3, 4, 5, 7]]).all() and np.isfinite(got[case.first[2] + 3]).all()


def test_rows_and_scales_far_from_one():
    """Rows of q of all magnitudes, scales of keys and values that differ by powers of ten between pages and heads, and pages of zeros."""
    case = Case([(300, 2), (77, 1)], 16, 2, 128, 128, seed=15)
    rng = case.rng
    case.pool.ks[:] = np.float32(0.02) * (10.0 ** rng.integers(-3, 1, case.pool.ks.shape))
    case.pool.vs[:] = np.float32(0.02) * (10.0 ** rng.integers(-6, 7, case.pool.vs.shape))
    case.pool.vs[case.table[case.order[0], 3]] = 0
    case.pool.ks[case.table[case.order[0], 5]] = 0
    cache = case.upload()
    q = rng.standard_normal((3, 8, 128))
    q *= 10.0 ** np.arange(-7, 1)[None, :, None]
    q[1, 2] = 0
    q = q.astype(np.float32).astype(np.float64)
    for factor, scale in ((1.0, 0.088), (1e-30, 0.088 * 1e30), (1e30, 0.088e-30)):
        x = np.float32(q * factor).astype(np.float64)
        got, _ = attend(case, cache, x, "f32", 8, scale)
        compare(case, x, "f32", 8, scale, got)


def test_the_same_call_gives_the_same_bits():
    case = Case([(700, 1), (3000, 2), (5, 1)], 16, 2, 128, 128, seed=16)
    cache = case.upload()
    q = case.rng.standard_normal((4, 8, 128)).astype(np.float32)
    a, _ = attend(case, cache, q, "f32", 8, 0.088)
    ws = None
    for _ in range(3):
        b, _ = attend(case, cache, q, "f32", 8, 0.088, ws=ws)
        assert (a == b).all()


def test_a_workspace_serves_any_shape_after_another():
    one = Case([(4000, 1)], 16, 2, 128, 128, seed=17)
    two = Case([(30, 1), (2000, 3)], 32, 4, 64, 64, seed=18)
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for case, n_head, scale in ((one, 8, 0.088), (two, 4, 0.125), (one, 16, 0.088), (two, 8, 0.125), (one, 8, 0.088)):
        cache = case.upload()
        q = case.rng.standard_normal((case.tokens, n_head, case.dim)).astype(np.float32).astype(np.float64)
        got, _ = attend(case, cache, q, "f32", n_head, scale, ws=ws)
        compare(case, q, "f32", n_head, scale, got)


def test_positions_far_beyond_32_bits_of_bytes():
    """A pool of 4.4 GB: pages at its end, and their neighbours untouched."""
    page, heads, dim = 128, 32, 256
    size = lib().b200_kv8_page_bytes(page, heads, dim, dim)
    n_pages = 4400 * (1 << 20) // size + 1
    pool = torch.zeros(n_pages, size, dtype=torch.uint8, device="cuda")
    case = Case([(0, 200)], page, heads, dim, dim, seed=19, spare=0)
    case.pool.put(np.zeros_like(case.pool.k), np.zeros_like(case.pool.v), np.zeros_like(case.pool.ks), np.zeros_like(case.pool.vs))
    case.upload()
    place = case.table[case.order[0], :2].copy()
    case.d_table[case.order[0], 0], case.d_table[case.order[0], 1] = n_pages - 1, n_pages - 3
    cache = Kv8Cache(pool.data_ptr(), n_pages, page, heads, dim, dim)
    k, v, tk, tv = rows_of(case, "bf16")
    run_store(case, cache, tk, tv, "bf16")
    reference_store(case, k, v)
    want = case.pool.records()
    end = case.pool.at[1] + 8 * heads
    assert (pool[n_pages - 1, :end].cpu().numpy() == want[place[0], :end]).all() and (pool[n_pages - 3, :end].cpu().numpy() == want[place[1], :end]).all()
    assert int(pool[:n_pages - 3].sum(dtype=torch.int64)) == 0 and int(pool[n_pages - 2].sum(dtype=torch.int64)) == 0
    q = rounded(case.rng.standard_normal((200, heads, dim)), "bf16")
    got, _ = attend(case, cache, q, "bf16", heads, 0.0625)
    compare(case, q, "bf16", heads, 0.0625, got)


# ------------------------------------------------------------------------------------------------ pages
class Device:
    """R.Pages on the GPU, beside pools whose records are compared whole."""

    def __init__(self, n_rows, stride, n_pages, page=16, shapes=((2, 64, 64), (1, 16, 32)), seed=0):
        self.ref = R.Pages(n_rows, stride, n_pages, page)
        self.table, self.len, self.refs = dev(self.ref.table), dev(self.ref.len), dev(self.ref.refs)
        self.map = Kv8Map(self.table.data_ptr(), stride, self.len.data_ptr(), self.refs.data_ptr(), n_rows, n_pages, page)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.pools = [torch.randint(0, 256, (n_pages, lib().b200_kv8_page_bytes(page, *s)), dtype=torch.uint8, device="cuda", generator=g) for s in shapes]
        self.want = [p.cpu().numpy().copy() for p in self.pools]
        self.caches = (Kv8Cache * max(1, len(shapes)))(*[Kv8Cache(p.data_ptr(), n_pages, page, *s) for p, s in zip(self.pools, shapes)])
        self.ws = torch.zeros(max(lib().b200_kv8_compact_workspace_bytes(n_pages), lib().b200_kv8_grow_workspace_bytes(1024)), dtype=torch.uint8, device="cuda")
        self.refused, self.live = ints(0), ints(-1)
        self.count = 0

    def same(self):
        for got, want, name in ((self.table, self.ref.table, "table"), (self.len, self.ref.len, "len"), (self.refs, self.ref.refs, "refs")):
            assert (got.cpu().numpy() == want).all(), name
        assert int(self.refused) == self.count
        for p, w in zip(self.pools, self.want):
            assert (p.cpu().numpy() == w).all()

    def moved(self, pairs):
        for w in self.want:
            before = w.copy()
            for a, b in pairs:
                w[b] = before[a]

    def cut(self, rows, keep=None, stream=None):
        r, k = ints(*rows), None if keep is None else ints(*keep)
        check(lib().b200_op_kv8_cut(C.byref(self.map), r.data_ptr(), None if k is None else k.data_ptr(), len(rows), stream))
        self.ref.cut(rows, keep)
        self.same()

    def fork(self, src, dst):
        s, d = ints(*src), ints(*dst)
        check(lib().b200_op_kv8_fork(C.byref(self.map), s.data_ptr(), d.data_ptr(), len(src), self.refused.data_ptr(), None))
        self.count += self.ref.fork(src, dst)
        self.same()

    def grow(self, rows, new):
        r, m, info = ints(*rows), ints(*new), torch.full((4, len(rows)), -9, dtype=torch.int32, device="cuda")
        check(lib().b200_op_kv8_grow(C.byref(self.map), self.caches, len(self.pools), r.data_ptr(), m.data_ptr(), len(rows), info.data_ptr(), self.refused.data_ptr(), self.ws.data_ptr(),
                                     self.ws.numel(), None))
        want, refused, copies = self.ref.grow(rows, new)
        self.count += refused
        self.moved(copies)
        assert (info.cpu().numpy() == want).all()
        self.same()

    def compact(self):
        check(lib().b200_op_kv8_compact(C.byref(self.map), self.caches, len(self.pools), self.live.data_ptr(), self.ws.data_ptr(), self.ws.numel(), None))
        n, moves = self.ref.compact()
        self.moved(moves)
        assert int(self.live) == n
        self.same()


def test_pages_by_hand():
    d = Device(8, 6, 20)
    d.grow([2, 5], [20, 16])
    d.fork([2, 2, 5], [0, 1, 3])
    d.grow([0, 1, 2], [1, 0, 13])       # row 0 copies its last page; row 1 asks for nothing; row 2 copies and needs one more
    d.grow([3], [1])                     # a full last page: nothing is copied
    d.cut([2, 0, 2, -1, 99], [17, 0, 0, 0, 0])
    d.cut([1])
    d.cut([5], [-3])
    d.compact()
    d.compact()


def test_pages_refusals():
    d = Device(6, 4, 10)
    d.grow([0, 0, 1, -1, 6, 2], [5, 5, 65, 1, 1, -1])      # named twice, beyond the table, no such row, negative
    d.fork([0, 0, 0, 7, 0, 2, 1], [1, 1, 0, 3, -1, 4, 5])  # named twice, onto itself, no such row; empty rows may be forked
    d.fork([1, 0], [3, 1])                                   # 1 is a dst of the call (and holds something)
    d.grow([2, 3, 4, 5], [64, 64, 33, 1])                    # 9 pages are left: 4, then 4, then 3 do not reach, and for the last neither
    d.grow([4, 5], [16, 1])                                  # one is left: the first gets it
    d.grow([5, 0], [0, 11])                                  # no page is needed
    d.compact()


def test_pages_without_caches_and_with_many():
    d = Device(4, 4, 9, shapes=())
    d.grow([0], [20])
    d.fork([0], [1])
    d.grow([1], [3])
    d.compact()
    d = Device(4, 4, 9, shapes=((1, 16, 16),) * 131)  # more than one launch takes
    d.grow([0, 1], [20, 7])
    d.fork([0], [2])
    d.grow([2, 0], [3, 1])
    d.cut([1])
    d.compact()


@pytest.mark.parametrize("seed", range(6))
def test_pages_through_many_calls(seed):
    """Calls at random over a pool that is too small at times; sizes around one round of the scans (8192 and 4096 pages) among them."""
    rng = np.random.default_rng(seed)
    n_pages = [40, 300, 4096, 9000, 16500, 700][seed]
    n_rows = [7, 60, 300, 1024, 500, 90][seed]
    page, stride = [16, 32, 16, 64, 16, 128][seed], [12, 30, 40, 25, 80, 33][seed]
    d = Device(n_rows, stride, n_pages, page, shapes=((1, 16, 16),), seed=seed)
    for _ in range(14):
        what = rng.choice(["grow", "grow", "grow", "fork", "cut", "compact"])
        n = int(rng.integers(1, min(n_rows, 1024) + 1))
        rows = rng.permutation(n_rows)[:n].tolist()
        if rng.random() < 0.3:
            rows[int(rng.integers(n))] = int(rng.choice([-1, n_rows, rows[0]]))
        if what == "grow":
            most = int(rng.choice([1, 5, page * 3, page * stride // 2]))
            d.grow(rows, [int(rng.integers(0, most + 1)) for _ in rows])
        elif what == "cut":
            d.cut(rows, None if rng.random() < 0.3 else [int(rng.integers(-1, page * stride)) for _ in rows])
        elif what == "fork":
            src = rng.integers(0, n_rows, n).tolist()
            d.fork(src, rows)
        else:
            d.compact()


def test_compaction_of_full_empty_and_single_pools():
    for n_pages in (1, 2, 17, 4096, 4097, 8200):
        d = Device(3, n_pages, n_pages, shapes=((1, 16, 16),))
        d.compact()                                    # nothing is live
        d.grow([1], [16 * n_pages])
        d.compact()                                    # everything is
        d.fork([1], [2])
        d.cut([1, 2], [0, 16 * (n_pages // 2)])
        d.compact()


def test_entries_that_no_window_reaches_may_be_taken_out():
    d = Device(3, 8, 12)
    d.grow([0, 1], [70, 40])
    for row, e in ((0, 0), (0, 2)):
        p = int(d.ref.table[row, e])
        d.ref.table[row, e], d.ref.refs[p] = -1, d.ref.refs[p] - 1
        d.table[row, e] = -1
        d.refs[p] -= 1
    d.fork([0], [2])
    d.grow([2, 0], [1, 60])
    d.compact()
    d.cut([0], [20])
    d.cut([2, 0])


def test_copies_of_pages():
    d = Device(2, 4, 30, shapes=((2, 64, 64), (3, 16, 48)))
    src, dst = ints(0, 5, 9, -1, 3, 30), ints(1, 6, 20, 2, -1, 4)
    check(lib().b200_op_kv8_copy_pages(d.caches, 2, src.data_ptr(), dst.data_ptr(), 6, None))
    d.moved([(0, 1), (5, 6), (9, 20)])
    d.same()


# ------------------------------------------------------------------------------------------------ together
class Serving:
    """Rows that grow, branch, are cut back and compacted, beside the values that each should hold."""

    def __init__(self, n_rows=6, n_pages=40, page=16, heads=2, dim=64, vdim=64, n_head=4, stream=None):
        self.n_rows, self.n_pages, self.page, self.heads, self.dim, self.vdim, self.n_head, self.stream = n_rows, n_pages, page, heads, dim, vdim, n_head, stream
        self.stride = n_pages
        self.d = Device(n_rows, self.stride, n_pages, page, shapes=((heads, dim, vdim),))
        self.pool = R.Pool(n_pages, page, heads, dim, vdim)
        raw = self.pool.records()
        self.d.pools[0].copy_(torch.from_numpy(raw))
        self.d.want[0][:] = raw
        self.rng = np.random.default_rng(1)

    def step(self, rows, new):
        """grow, store, attend: the results, compared with the reference's."""
        d, n, tokens = self.d, len(rows), sum(new)
        r, m, info = ints(*rows), ints(*new), torch.zeros(4, n, dtype=torch.int32, device="cuda")
        k, v, q = (self.rng.standard_normal((tokens, h, s)).astype(np.float32) for h, s in ((self.heads, self.dim), (self.heads, self.vdim), (self.n_head, self.dim)))
        tk, tv, tq = (dev(x.reshape(tokens, -1)) for x in (k, v, q))
        out = torch.zeros(tokens, self.n_head * self.vdim, device="cuda")
        where = (info.data_ptr(), d.table.data_ptr(), self.stride, self.n_rows, n, tokens)
        store = Kv8StoreArgs(d.caches[0], tk.data_ptr(), tk.stride(0), tv.data_ptr(), tv.stride(0), *where, L.F32)
        attn = Kv8AttnArgs(d.caches[0], tq.data_ptr(), tq.stride(0), out.data_ptr(), out.stride(0), *where, max(new), self.n_head, L.F32, None, 0, 0, 0.125, 0.0, 0)
        ws = torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(attn)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        check(lib().b200_op_kv8_grow(C.byref(d.map), d.caches, 1, r.data_ptr(), m.data_ptr(), n, info.data_ptr(), d.refused.data_ptr(), d.ws.data_ptr(), d.ws.numel(), self.stream))
        check(lib().b200_op_kv8_store(C.byref(store), self.stream))
        check(lib().b200_op_kv8_attn(C.byref(attn), ws.data_ptr(), ws.numel(), self.stream))
        torch.cuda.synchronize()
        _, refused, copies = d.ref.grow(rows, new)
        assert refused == 0
        self.copy(copies)
        got, at = out.double().cpu().numpy().reshape(tokens, self.n_head, self.vdim), 0
        for row, c in zip(rows, new):
            held, entries = int(d.ref.len[row]) - c, d.ref.table[row]
            self.pool.store(entries, k[at:at + c], v[at:at + c], held)
            if c:
                want, mass, size = self.pool.attend(entries, q[at:at + c], held, 0.125)
                assert (np.abs(got[at:at + c] - want) <= bound("f32", mass, size, want, 0)).all()
            at += c
        d.want[0][:] = self.pool.records()
        d.same()

    def copy(self, pairs):
        for x in (self.pool.k, self.pool.v, self.pool.ks, self.pool.vs, self.pool.raw):
            before = x.copy()
            for a, b in pairs:
                x[b] = before[a]

    def compact(self):
        before = self.d.ref.table.copy(), self.d.ref.refs.copy()
        _, moves = R.Pages.compact(self.d.ref)
        self.d.ref.table, self.d.ref.refs = before
        self.copy(moves)
        self.d.compact()


def serve(s):
    s.step([0, 3], [37, 1])               # a prompt and a short one
    s.step([0, 3], [1, 1])
    s.d.fork([0, 0, 3], [1, 2, 4])        # branches share all pages
    s.step([1, 2, 0, 4], [1, 1, 1, 2])    # each writes to a copy of the last page
    s.step([2, 1], [20, 3])
    s.d.cut([0, 2], [0, 45])              # one ends, one drops what was rejected
    s.compact()
    s.step([1, 2, 3, 4, 0], [1, 4, 1, 0, 18])
    s.d.cut([1, 2, 3, 4])
    s.compact()
    s.step([0], [1])


def test_serving():
    serve(Serving())


def test_serving_on_another_stream():
    stream = torch.cuda.Stream()
    s = Serving(page=32, dim=128, vdim=96, stream=stream.cuda_stream)
    for rows, new in (([0, 2], [40, 3]), ([2, 0], [1, 1]), ([0, 1, 2], [1, 70, 1])):
        s.step(rows, new)


def test_captured_step():
    """cut, grow, store, attend as a graph that is replayed: every replay finds the lengths that the one before left."""
    s = Serving(n_rows=3, n_pages=20)
    s.step([0, 1, 2], [20, 3, 16])
    d, rows, one = s.d, ints(0, 1, 2), ints(1, 1, 1)
    info = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    tk, tv, tq, out = torch.zeros(3, 128, device="cuda"), torch.zeros(3, 128, device="cuda"), torch.zeros(3, 256, device="cuda"), torch.zeros(3, 256, device="cuda")
    where = (info.data_ptr(), d.table.data_ptr(), s.stride, 3, 3, 3)
    store = Kv8StoreArgs(d.caches[0], tk.data_ptr(), 128, tv.data_ptr(), 128, *where, L.F32)
    attn = Kv8AttnArgs(d.caches[0], tq.data_ptr(), 256, out.data_ptr(), 256, *where, 1, 4, L.F32, None, 0, 0, 0.125, 0.0, 0)
    ws = torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(attn)), dtype=torch.uint8, device="cuda")
    stream = C.c_void_p()
    check(lib().b200_stream_create(C.byref(stream)))
    torch.cuda.synchronize()
    check(lib().b200_graph_begin_capture(stream))
    check(lib().b200_op_kv8_grow(C.byref(d.map), d.caches, 1, rows.data_ptr(), one.data_ptr(), 3, info.data_ptr(), None, d.ws.data_ptr(), d.ws.numel(), stream))
    check(lib().b200_op_kv8_store(C.byref(store), stream))
    check(lib().b200_op_kv8_attn(C.byref(attn), ws.data_ptr(), ws.numel(), stream))
    graph = C.c_void_p()
    check(lib().b200_graph_end_capture(stream, C.byref(graph)))
    for _ in range(40):  # across page borders
        k, v, q = (s.rng.standard_normal((3, h, 64)).astype(np.float32) for h in (2, 2, 4))
        for t, x in ((tk, k), (tv, v), (tq, q)):
            t.copy_(torch.from_numpy(x.reshape(3, -1)))
        torch.cuda.synchronize()
        check(lib().b200_graph_launch(graph, stream))
        check(lib().b200_stream_synchronize(stream))
        _, refused, copies = d.ref.grow([0, 1, 2], [1, 1, 1])
        assert refused == 0 and not copies
        got = out.double().cpu().numpy().reshape(3, 4, 64)
        for i in range(3):
            held, entries = int(d.ref.len[i]) - 1, d.ref.table[i]
            s.pool.store(entries, k[i:i + 1], v[i:i + 1], held)
            want, mass, size = s.pool.attend(entries, q[i:i + 1], held, 0.125)
            assert (np.abs(got[i:i + 1] - want) <= bound("f32", mass, size, want, 0)).all()
    d.want[0][:] = s.pool.records()
    d.same()
    check(lib().b200_graph_destroy(graph))
    check(lib().b200_stream_destroy(stream))
