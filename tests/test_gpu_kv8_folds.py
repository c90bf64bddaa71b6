"""Prompts of 16 bits behind so many keys that their sums are folded (more than 4096 with f16 rows, 8192 with bf16), where each block of rows is one CTA's: against tests/kv8_ref.py with the bounds
of test_gpu_kv8.py, which hold for sums of any length once they are folded (2^-15 of the mass leaves room for 512 additions of 2^-24)."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import Case, attend, rounded
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
