"""tests/state_stretches.py on the CPU: it says what tests/state_ref.py says, and its tolerances notice sums of d that are a little wrong."""
import numpy as np
import pytest

import state_ref as R
import state_stretches as S


def made(rows, seed=0, ch=6, n=4):
    rng = np.random.default_rng(seed)
    return dict(x=rng.normal(size=(rows, ch)), raw=rng.normal(size=(rows, ch)) * 1.5 - 2, b=rng.normal(size=(rows, n)), c=rng.normal(size=(rows, n)), a=-np.exp(rng.normal(size=(ch, n)) - 5),
                state=rng.normal(size=(ch, n)))


@pytest.mark.parametrize("rows,stretch", [(300, 64), (128, 64), (64, 64), (65, 64)])
def test_it_is_the_scan(rows, stretch):
    m = made(rows)
    y, h, tol, _ = S.scan(**m, stretch=stretch)
    want, state, wide, _ = R.scan(m["x"], m["raw"], m["b"], m["c"], None, m["a"], None, None, [[0], [rows], [0], [0]], m["state"][None], True, np.zeros_like(y), "f32")
    assert np.allclose(y, want, rtol=1e-11, atol=1e-12) and np.allclose(h, state[0], rtol=1e-11)
    assert (tol < 3 * wide).all()


def f32_sum(d):
    """Row by row in groups of 16, each group's sum and the whole in f32."""
    total = np.zeros(d.shape[1], np.float32)
    for i in range(0, len(d), 16):
        some = d[i].astype(np.float32)
        for row in d[i + 1:i + 16].astype(np.float32):
            some = some + row
        total = total + some
    return total.astype(np.float64)


def f64_sum(d):
    total = np.zeros(d.shape[1])
    for i in range(0, len(d), 16):
        some = d[i].astype(np.float32)
        for row in d[i + 1:i + 16].astype(np.float32):
            some = some + row
        total = total + some
    return total.astype(np.float32).astype(np.float64)


LONG = 4096


@pytest.mark.parametrize("sum_of,found", [(f64_sum, False), (f32_sum, True), (lambda d: d.sum(0) * (1 + 2.0 ** -14), True), (lambda d: d.sum(0) * (1 + 2.0 ** -16), True), (lambda d: d[:-1].sum(0), True)])
def test_sums_that_are_a_little_wrong_are_noticed(sum_of, found):
    """Long stretches of a state that only fades, where nothing but the carrying adds errors: what one rounding leaves is inside the tolerance, a sum kept in f32 is not."""
    d, a = S.fading(LONG, 8, 4, 2.0, seed=1)
    steps = np.tile(d, (LONG, 1))
    wrong = right = np.ones((8, 4))
    tol = np.zeros((8, 4))
    for _ in range(31):
        tol = tol * np.exp(steps.sum(0)[:, None] * a) + S.carry_error(right, steps.sum(0)[:, None] * a)
        right, wrong = right * np.exp(steps.sum(0)[:, None] * a), wrong * np.exp(sum_of(steps)[:, None] * a)
    assert (np.abs(wrong - right) > tol).any() == found


@pytest.mark.parametrize("by,found", [(0.0, False), (2.0 ** -11, True)])
def test_ordinary_rows(by, found):
    """The same for rows as a layer has them, whose own errors are the larger part of the tolerance."""
    m = made(3000, ch=8, n=4)
    m["raw"], m["a"] = np.abs(m["raw"]) * 0.05, -np.random.default_rng(1).uniform(0.05, 0.2, (8, 4))
    y, _, tol, _ = S.scan(**m, stretch=96, is_softplus=False)
    wrong = S.scan(**m, stretch=96, sum_of=lambda d: d.sum(0) * (1 + by), is_softplus=False)[0]
    assert (np.abs(wrong - y) > tol).any() == found
