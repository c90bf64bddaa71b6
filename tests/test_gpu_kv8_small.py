"""Stores under the smallest scales that a page may have, against tests/kv8_ref.py bit by bit: from 2^-126 to 2^-125 half a step is no f32."""
import numpy as np
import pytest

from test_gpu_kv8 import Case, dev, reference_store, run_store

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -149


def loudest(steps):
    """The f32 value (in units of 2^-149) whose 127th part, rounded, is `steps` units."""
    x = np.float32(127 * np.float64(steps) * UNIT)
    assert np.float32(np.float64(x) / 127) == np.float32(steps * UNIT)
    return x


@pytest.mark.parametrize("steps", [2 ** 23, 2 ** 23 + 1, 10905191, 10905193, 11184809, 13421773, 2 ** 24 - 1])
@pytest.mark.parametrize("name", ["f32"])
def test_store_beside_half_a_step(steps, name):
    case = Case([(0, 16)], heads=1, dim=256, vdim=256, seed=6)
    cache = case.upload()
    n = np.arange(-126, 126, dtype=np.float64)
    half = n * steps + steps / 2
    x = np.zeros((16, 1, 256), np.float32)
    for t, add in enumerate((0.5, -0.5, 0.0, 1.5, -1.5)):  # units beside half a step; rounded where f32 has no such value
        x[t, 0, :252] = np.float32((half + add) * UNIT)
    x[:, 0, 255] = loudest(steps)
    x[5:10, 0, :252] = np.nextafter(x[:5, 0, :252], np.float32(1))
    x[10:15, 0, :252] = np.nextafter(x[:5, 0, :252], np.float32(-1))
    v = x[::-1].copy()
    run_store(case, cache, dev(x.reshape(16, -1)), dev(v.reshape(16, -1)), name)
    reference_store(case, x.astype(np.float64), v.astype(np.float64))
    assert case.pool.ks[case.table[case.order[0], 0], 0] == np.float32(steps * UNIT)
    case.same_pool()


@pytest.mark.parametrize("first,then", [(2 ** 23 + 1, 10905191), (2 ** 23 + 3, 13421773), (9000001, 2 ** 24 - 1), (8400001, 12600003)])
def test_what_a_page_held_follows(first, then):
    """All ints of a page under a scale that grows to another one of that range."""
    case = Case([(0, 2)], heads=1, dim=256, vdim=256, seed=7)
    cache = case.upload()
    x = np.zeros((2, 1, 256), np.float32)
    x[0, 0, :255] = np.float32(np.arange(-127, 128) * np.float64(first) * UNIT)
    x[1, 0] = np.float32(np.arange(-128, 128) / 3 * np.float64(first) * UNIT)
    x[0, 0, 255] = loudest(first)
    run_store(case, cache, dev(x.reshape(2, -1)), dev(x.reshape(2, -1)), "f32")
    reference_store(case, x.astype(np.float64), x.astype(np.float64))
    case.same_pool()
    case.seqs, case.new, case.tokens = [(2, 1)], [1], 1
    case.d_info = case.info()
    y = np.zeros((1, 1, 256), np.float32)
    y[0, 0, 3] = loudest(then)
    run_store(case, cache, dev(y.reshape(1, -1)), dev(y.reshape(1, -1)), "f32")
    reference_store(case, y.astype(np.float64), y.astype(np.float64))
    assert case.pool.ks[case.table[case.order[0], 0], 0] == np.float32(then * UNIT)
    case.same_pool()
