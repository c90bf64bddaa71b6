"""Precision of attention over the paged 8-bit cache (include/b200_kv8.h) where the length of sums shows, against softmax in 64 bits on the GPU.

Keys are made so that scores are exact or hardly matter, values have scales that are powers of two (but in "inexact") and enter exactly as they are; what is left is how sums are taken.
Kinds of rows (keys a query sees: key 0 and n others):
  "even"     all weights are 1, values of one sign: sums grow evenly, and are exact until they pass 24 bits
  "inexact"  the same under a scale of 22 bits: every addition has bits to lose
  "zero"     all weights are 1, values around zero
  "first"    key 0 takes all the weight (the others e^-30 of it): what comes behind it must not change its value
  "small"    key 0 has most of the weight, each other about 2^-20 of it
"""
import ctypes as C
import math

import pytest
import torch

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Kv8AttnArgs, Kv8Cache, check, lib

pytestmark = pytest.mark.gpu

TYPES = {"f32": (L.F32, torch.float32), "f16": (L.F16, torch.float16), "bf16": (L.BF16, torch.bfloat16)}
KINDS = ["even", "inexact", "zero", "first", "small"]
V_SCALE = 2.0 ** -7
INEXACT = 2905413 * 2.0 ** -28  # 0.0108


class Rows:
    """n_seq sequences that share the pages of `n` tokens, the last `new` of which ask."""

    def __init__(self, kind, n_seq, n, new, heads, dim, vdim, page=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.n_seq, self.n, self.new, self.heads, self.dim, self.vdim, self.page = n_seq, n, new, heads, dim, vdim, page
        n_pages = -(-n // page)
        rand = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda").to(torch.int8)  # noqa: E731
        self.v = rand(1, 128, n_pages * page, heads, vdim) if kind in ("even", "inexact") else rand(-127, 128, n_pages * page, heads, vdim)
        self.v[0] = rand(60, 128, heads, vdim)
        self.v_scale = INEXACT if kind == "inexact" else V_SCALE
        if kind in ("even", "inexact", "zero"):
            self.k = torch.zeros(n_pages * page, heads, dim, dtype=torch.int8, device="cuda")
            self.scale = 1.0
        else:  # q = 1: scores are scale times the sum of a key's ints
            self.k = rand(-127, -100, n_pages * page, heads, dim)
            self.k[0] = 127
            self.scale = (30 if kind == "first" else 20 * math.log(2)) / (240.0 * dim)
        nk, nv = heads * page * dim, heads * page * vdim
        pool = torch.zeros(n_pages, lib().b200_kv8_page_bytes(page, heads, dim, vdim), dtype=torch.uint8, device="cuda")
        pool[:, :nk] = self.k.reshape(n_pages, page, heads, dim).transpose(1, 2).reshape(n_pages, nk).view(torch.uint8)
        pool[:, nk:nk + nv] = self.v.reshape(n_pages, page, heads, vdim).transpose(1, 2).reshape(n_pages, nv).view(torch.uint8)
        pool[:, nk + nv:nk + nv + 8 * heads] = torch.tensor([1.0] * heads + [self.v_scale] * heads, device="cuda").view(torch.uint8)
        self.pool = pool
        self.cache = Kv8Cache(pool.data_ptr(), n_pages, page, heads, dim, vdim)
        self.table = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).to("cuda", torch.int32)
        pool[self.table.long()] = pool.clone()
        self.table = self.table.repeat(n_seq, 1).contiguous()
        self.info = torch.tensor([[i * new for i in range(n_seq)], [new] * n_seq, list(range(n_seq)), [n - new] * n_seq], dtype=torch.int32, device="cuda")

    def run(self, name, n_head, q=None, scale=None, f16=0, max_new=0, **opt):
        """[n_seq][new][n_head][vdim] in 64 bits"""
        tokens, (code, dtype) = self.n_seq * self.new, TYPES[name]
        q = torch.ones(tokens, n_head * self.dim, dtype=dtype, device="cuda") if q is None else q
        out = torch.full((tokens, n_head * self.vdim), math.nan, dtype=dtype, device="cuda")
        a = Kv8AttnArgs(self.cache, q.data_ptr(), n_head * self.dim, out.data_ptr(), n_head * self.vdim, self.info.data_ptr(), self.table.data_ptr(), self.table.shape[1], self.n_seq, self.n_seq, tokens,
                        max_new or self.new, n_head, code, None, opt.get("window", 0), 0, self.scale if scale is None else scale, opt.get("softcap", 0.0), f16)
        ws = torch.zeros(lib().b200_kv8_attn_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
        for _ in range(2):  # (the workspace serves one call after the other)
            check(lib().b200_op_kv8_attn(C.byref(a), ws.data_ptr(), ws.numel(), None))
        torch.cuda.synchronize()
        return out.double().reshape(self.n_seq, self.new, n_head, self.vdim)

    def want(self, token):
        """What new token number `token` of a sequence gets, [heads][vdim], and the mass of what it sums."""
        n = self.n - self.new + token + 1
        s = self.k[:n].double().sum(-1) * float(torch.tensor(self.scale, dtype=torch.float32))
        p = torch.softmax(s, dim=0)
        v = self.v[:n].double() * self.v_scale
        return torch.einsum("nh,nhd->hd", p, v), torch.einsum("nh,nhd->hd", p, v.abs())


def off(got, want, mass):
    """Errors relative to the mass."""
    return (got - want) / mass


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_seq,n,heads,n_head,vdim,f16", [(64, 32000, 8, 32, 128, 0), (64, 32000, 8, 16, 64, 0), (40, 32000, 8, 8, 256, 0), (64, 32000, 8, 32, 128, 1), (3, 131000, 1, 5, 128, 0)])
def test_long_sums_of_few_rows(kind, n_seq, n, heads, n_head, vdim, f16):
    """Single tokens of many sequences: whole blocks, or long runs of them, fall to one CTA.
    A warp takes 32 keys at a time, every fourth such tile.  A tile's products are at most four additions on the tensor cores, each cutting off less than 2^-23 of the tile's mass: 2^-21.  Tiles are
    added in f32, to the nearest: N = n / 128 + 8 roundings of half a last place, 2^-24 of the sum, either way, 6 standard deviations of 2^-24 sqrt(N / 3).  Weights: 2^-22 of two f16 (they are powers of two
    times 1 in "even" and "zero"; with one f16 each of the small ones is off by 2^-12, and their sum by 2^-12 of its share of the mass), exponentials 2^-21; the sum of the weights as
    the tiles' sums.  In "first" additions behind the first tile are of nothing: no term in N."""
    if kind in ("small", "inexact") and f16:
        pytest.skip("weights are rounded to f16 there")
    r = Rows(kind, n_seq, n, 1, heads, 16, vdim, seed=n_head)
    want, mass = (x.repeat_interleave(n_head // heads, dim=0) for x in r.want(0))
    e = off(r.run("f32", n_head, f16=f16), want, mass)
    assert not e.isnan().any()
    many = 0.0 if kind == "first" else 2 * 6 * 2.0 ** -24 * math.sqrt((n / 128 + 8) / 3)
    assert e.abs().max() <= 2.0 ** -21 + 2.0 ** -20 + many, float(e.abs().max())


PROMPTS = [  # heads, n_head, new: two groups of rows a CTA; one; several CTAs a block
    (40, 40, 520), (20, 20, 520), (4, 64, 64)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,n_head,new", PROMPTS)
def test_long_sums_of_prompts(kind, heads, n_head, new):
    """f32 rows.  Between two folds 128 additions, each cutting off less than 2^-23 of the sum so far: 2^-17 of a sum that grows evenly; where all the weight is on key 0 later additions are of
    nothing.  Folds and the sum of weights are roundings to the nearest, N = n / 64 of them, as above; weights and exponentials as above."""
    n = 30000
    r = Rows(kind, 1, n, new, heads, 16, 64, seed=new)
    got = r.run("f32", n_head)
    for token in (0, 1, new // 2, new - 1):
        want, mass = (x.repeat_interleave(n_head // heads, dim=0) for x in r.want(token))
        e = off(got[0, token], want, mass)
        many = 0.0 if kind == "first" else 2.0 ** -17 + 6 * 2.0 ** -24 * math.sqrt(n / 64 / 3)
        assert not e.isnan().any() and e.abs().max() <= 2.0 ** -20 + many, (token, float(e.abs().max()))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_head,new", PROMPTS)
def test_long_sums_of_prompts_of_16_bits(name, heads, n_head, new):
    """100,000 keys.  Sums cut off less than 2^-23 of themselves in each of at most 512 additions between two folds: 2^-15 of sums that grow evenly, far below half a step of f16.  Weights and
    exponentials 2^-20.  Rounding is monotone: what is off by a share d of itself before it is rounded lies between the roundings of 1 - d and 1 + d times the exact result."""
    n, dtype = 100000, TYPES[name][1]
    r = Rows("first", 1, n, new, heads, 16, 64, seed=new)
    got = r.run(name, n_head)[0]
    assert (got == (r.v[0].double() * V_SCALE).repeat_interleave(n_head // heads, dim=0)).all()  # ints of 7 bits: both types hold them
    r = Rows("even", 1, n, new, heads, 16, 64, seed=new)
    got = r.run(name, n_head)[0]
    v = r.v.double() * V_SCALE
    sums = v[:n - new].sum(0) + v[n - new:n].cumsum(0)
    want = (sums / torch.arange(n - new + 1, n + 1, device="cuda")[:, None, None]).repeat_interleave(n_head // heads, dim=1)
    d = 2.0 ** -15 + 2.0 ** -20
    lo, hi = ((want * (1 + x)).to(dtype).double() for x in (-d, d))
    assert ((got >= lo) & (got <= hi)).all()


@pytest.mark.parametrize("cap", [4.0, 30.0, 50.0])
@pytest.mark.parametrize("n_seq,new,heads,n_head,dim,vdim", [(4, 1, 8, 32, 64, 64), (1, 7, 8, 24, 128, 80), (2, 4, 1, 4, 192, 256), (1, 520, 40, 40, 64, 64), (3, 129, 4, 40, 128, 128)])
def test_soft_cap_of_f32_rows(n_seq, new, heads, n_head, dim, vdim, cap):
    """Every query sees two keys, whose values are v and -v: what comes out is v tanh(d / 2) of the difference d of their scores s.
    q has 8 bits and keys 8, so products and their sums are exact in f32.  s / cap takes four roundings (2^-22 of it), tanh two units in the last place (2^-22), the way back to a score and its difference
    from the maximum three roundings (below 2^-22 of the largest score), the exponential 2^-22 of itself, weights, their sum and the quotient 2^-21: with both scores, 2 p (1 - p) <= 1/2,
    v (|s1| + |s2|) 2^-21 + 2^-20 v."""
    r = Rows("zero", n_seq, 300 + new, new, heads, dim, vdim, page=32, seed=int(cap))
    g = torch.Generator(device="cuda").manual_seed(dim)
    n_pages, page = r.pool.shape[0], r.page
    sign = torch.where(torch.arange(n_pages * page, device="cuda") % 2 == 0, 1, -1).to(torch.int8)
    k = torch.randint(-127, 128, (n_pages * page, heads, dim), generator=g, device="cuda").to(torch.int8)
    v = sign[:, None, None] * torch.randint(60, 128, (1, heads, vdim), generator=g, device="cuda").to(torch.int8)
    nk, nv = heads * page * dim, heads * page * vdim
    at = r.table[0].long()
    r.pool[at, :nk] = k.reshape(n_pages, page, heads, dim).transpose(1, 2).reshape(n_pages, nk).view(torch.uint8)
    r.pool[at, nk:nk + nv] = v.reshape(n_pages, page, heads, vdim).transpose(1, 2).reshape(n_pages, nv).view(torch.uint8)
    q = torch.randint(-127, 128, (n_seq, new, n_head, dim), generator=g, device="cuda").float() / 64
    scale = float(torch.tensor(0.7 / (math.sqrt(dim) * 73 * 1.15), dtype=torch.float32))
    got = r.run("f32", n_head, q=q.reshape(n_seq * new, -1).contiguous(), scale=scale, window=2, softcap=cap)
    pos = torch.arange(r.n - new, r.n, device="cuda")
    s = [cap * torch.tanh((q.double() * k[pos - i].double().repeat_interleave(n_head // heads, dim=1)).sum(-1) * scale / cap) for i in (0, 1)]
    own = v[pos].double().repeat_interleave(n_head // heads, dim=1) * V_SCALE
    want = own * torch.tanh((s[0] - s[1]) / 2)[..., None]
    most = own.abs() * ((s[0].abs() + s[1].abs()) * 2.0 ** -21 + 2.0 ** -20)[..., None]
    assert ((got - want).abs() <= most).all(), float(((got - want).abs() / most).max())


@pytest.mark.parametrize("kind", ["even", "zero", "first"])
@pytest.mark.parametrize("heads,n_head,new", PROMPTS)
def test_long_sums_of_prompts_with_f16_products(kind, heads, n_head, new):
    """f32 rows whose queries and weights (powers of two here) are one f16 each: 512 additions between two folds, 2^-15 of a sum that grows evenly; the rest as above."""
    n = 30000
    r = Rows(kind, 1, n, new, heads, 16, 64, seed=new)
    got = r.run("f32", n_head, f16=1)
    for token in (0, 1, new // 2, new - 1):
        want, mass = (x.repeat_interleave(n_head // heads, dim=0) for x in r.want(token))
        e = off(got[0, token], want, mass)
        many = 0.0 if kind == "first" else 2.0 ** -15 + 6 * 2.0 ** -24 * math.sqrt(n / 64 / 3)
        assert not e.isnan().any() and e.abs().max() <= 2.0 ** -20 + many, (token, float(e.abs().max()))
