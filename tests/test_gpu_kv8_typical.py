"""Errors of attention over the paged 8-bit cache as a whole, against tests/kv8_ref.py: tight where a bound for every single result (test_gpu_kv8.py) has to be wide.

Queries and keys are normal, scores have a deviation N of about 1, so that a query's weights are spread over sixteen keys and more.
f32 rows.  A score of 128 dims takes 16 additions of two terms on the tensor cores, each cutting off half of 2^-23 of what is summed up (2 N at most, on average): 2^-19 N; queries as two f16 leave
2^-23 of the largest over, 2^-21 N at most; factors and exponential 2^-21: 2^-18 in all.  A result is a mean of values, each off by that share of its weight, independent of the others but for what they have in
common, which the division takes out: 2^-18 / sqrt(16) = 2^-20 of the mass of a result, root mean square.  Sums behind up to 1330 keys cut off 2^-19 of a sum that grows evenly between two folds, and less around 0.
f16 rows.  Queries are exact, weights two f16: results before they are rounded are as above.  A result of mass M that is off by e = 2^-20 M is rounded to the other side with a probability of 2 e / step;
the mean of |e| is below its root mean square, so the expected count is below the sum of that; six deviations more at most.
"""
import numpy as np
import pytest

from test_gpu_kv8 import Case, attend, rounded

pytestmark = pytest.mark.gpu

STEPS = {"few": ([(700, 1), (300, 2), (1200, 1), (64, 3)], 24, 8), "prompt": ([(600, 130)], 32, 4), "ragged": ([(1200, 130), (0, 70), (64, 200)], 40, 20)}


def results(step, name, dim, vdim, seed, **opt):
    """(got, want, mass) of all tokens and of some heads, and the case."""
    seqs, n_head, heads = STEPS[step]
    case = Case(seqs, 16, heads, dim, vdim, seed=seed)
    cache = case.upload()
    q = rounded(case.rng.standard_normal((case.tokens, n_head, dim)) * 1.2, name)
    scale = dim ** -0.5
    got, _ = attend(case, cache, q, name, n_head, scale, **opt)
    group = n_head // heads
    some = [0, heads // 2, heads - 1]
    heads_of = [h * group + i for h in some for i in range(group)]
    case.pool.heads = len(some)
    case.pool.put(*(x[:, some] for x in (case.pool.k, case.pool.v, case.pool.ks, case.pool.vs)))
    want, mass = [], []
    for (held, m), r, f in zip(case.seqs, case.order, case.first):
        w, a, _ = case.pool.attend(case.table[r], q[f:f + m][:, heads_of], held, np.float64(np.float32(scale)))
        keep = np.arange(m) + held >= 64  # (the first tokens see few keys)
        want.append(w[keep]); mass.append(a[keep])
    here = np.concatenate([f + np.arange(m)[np.arange(m) + h >= 64] for (h, m), f in zip(case.seqs, case.first)])
    return got[here][:, heads_of], np.concatenate(want), np.concatenate(mass)


@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (96, 80), (256, 256)])
@pytest.mark.parametrize("step", STEPS)
def test_f32_rows(step, dim, vdim):
    got, want, mass = results(step, "f32", dim, vdim, dim)
    rms = float(np.sqrt(np.mean(((got - want) / mass) ** 2)))
    assert rms <= 2.0 ** -20, rms
    # queries and weights rounded to f16, as a caller may ask for, are what this test would notice
    got, want, mass = results(step, "f32", dim, vdim, dim, f16=1)
    assert 2.0 ** -18 < np.sqrt(np.mean(((got - want) / mass) ** 2)) < 2.0 ** -12


def share_of_others(x, want, mass):
    """How many results are not the exact one rounded to f16, and how many may not be."""
    nearest = want.astype(np.float16).astype(np.float64)
    step = np.spacing(np.abs(want).astype(np.float16)).astype(np.float64)
    expected = float((2 * 2.0 ** -20 * mass / step).clip(max=1).sum())
    return int((x != nearest).sum()), expected + 6 * expected ** 0.5


@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (96, 80), (256, 128)])
@pytest.mark.parametrize("step", STEPS)
def test_f16_rows(step, dim, vdim):
    got, want, mass = results(step, "f16", dim, vdim, dim)
    others, most = share_of_others(got, want, mass)
    assert others <= most, (others, most, want.size)
    # weights of one f16 each: off by 2^-12 / sqrt(3) of themselves, by 2^-13 of a result that is their mean
    planted = want * (1 + np.random.default_rng(1).standard_normal(want.shape) * 2.0 ** -13)
    assert share_of_others(planted.astype(np.float16).astype(np.float64), want, mass)[0] > most
