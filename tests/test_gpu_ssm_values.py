"""Scans on the GPU over values at the ends of their range: what is infinite by the definition is infinite, with its sign, and what is finite stays so."""
import numpy as np
import pytest

from test_gpu_ssm import Scan, run

pytestmark = pytest.mark.gpu


def defined(s):
    """dst and states by the definition, row by row in 64 bits: infinities and NaN as arithmetic makes them."""
    of = np.arange(s.ch) // (s.ch // s.groups)
    dst, state = s.dst.copy(), s.state.copy()
    with np.errstate(all="ignore"):
        for first, count, slot, begins in s.info.T.tolist():
            h = np.zeros_like(state[slot]) if begins else state[slot].copy()
            for t in range(first, first + count):
                d = s.dt[t] + (0 if s.bias is None else s.bias)
                if s.softplus:
                    d = np.maximum(d, 0) + np.log1p(np.exp(-np.abs(d)))
                h = np.exp(d[:, None] * s.a) * h + (d * s.x[t])[:, None] * s.b[t].reshape(s.groups, s.n)[of]
                y = (h * s.c[t].reshape(s.groups, s.n)[of]).sum(1)
                if s.skip is not None:
                    y = y + s.skip * s.x[t]
                dst[t] = y if s.z is None else y * (s.z[t] / (1 + np.exp(-s.z[t])))
            if count:
                state[slot] = h
    return dst, state


def kinds(v):
    return np.where(np.isnan(v), 3, np.where(np.isposinf(v), 1, np.where(np.isneginf(v), 2, 0)))


def same_kinds(s):
    want, state = defined(s)
    got, got_state = s.d["dst"].get(), s.d_state.get().reshape(state.shape)
    for g, w in ((got, want), (got_state, state)):
        off = kinds(g) != kinds(w)
        assert not off.any(), (int(off.sum()), np.argwhere(off)[:5].tolist(), g[off][:5].tolist(), w[off][:5].tolist())
    return got, want, got_state, state


SIZES = [1, 3, 4, 5, 7, 8, 11, 13, 16, 20, 29, 32, 41, 64, 67, 100, 127, 128]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("count", [1, 5, 40, 300])
def test_infinities_whatever_the_number_of_states(n, count):
    """Inputs and steps that are infinite, where all states of the channel go the same way: the result is infinite with a sign, not no number, also where d_state fills no register."""
    for gate, skip in ((False, False), (True, True)):
        s = Scan([(count, 1, False), (count, 0, True)], 40, n, "f32", gate=gate, skip=skip, seed=n, slow=True)
        s.b, s.c, s.state = np.abs(s.b) + 0.125, np.abs(s.c) + 0.125, np.abs(s.state)
        s.x[:, 30:] = np.abs(s.x[:, 30:]) + 0.125
        if gate:
            s.z = np.abs(s.z) + 0.125
            s.skip = np.abs(s.skip)
        t = count // 2
        s.x[t, 3], s.x[count + t, 5], s.x[t, 7] = np.inf, np.inf, -np.inf
        s.dt[t, 31], s.dt[count + t, 32] = np.inf, np.inf
        a = s.upload()
        a.max_new = count
        run(a)
        got = same_kinds(s)[0]
        assert np.isposinf(got[t:count, 3]).all() and np.isposinf(got[count + t:, 5]).all() and np.isneginf(got[t:count, 7]).all() and np.isposinf(got[t:count, 31]).all()


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("n", [5, 16, 40])
@pytest.mark.parametrize("count", [1, 3, 18, 50, 300])
def test_states_that_fade_at_once(n, count, softplus):
    """a of -inf, as a type of fewer bits or an overflowing exponential leaves it: the state is what the last row put there, also where a group of rows ends behind the sequence's last."""
    s = Scan([(count, 1, False), (count, 0, True)], 40, n, "f32", seed=n, softplus=softplus, slow=True)
    s.a[3] = -np.inf
    s.a[7, ::2] = -np.inf
    s.a[9] = -3.4028234663852886e38
    if not softplus:
        s.dt, s.bias = np.abs(s.dt) + 2.0 ** -20, np.abs(s.bias)
    a = s.upload()
    a.max_new = count
    run(a)
    got, want, got_state, state = same_kinds(s)
    assert np.isfinite(want).all() and np.allclose(got, want, rtol=1e-4, atol=1e-4) and np.allclose(got_state, state, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("n", [16, 40])
@pytest.mark.parametrize("count", [1, 3, 18])
def test_no_time_passes_with_a_step_of_nothing(n, count):
    """d of 0 leaves every state as it is, whatever its rate: infinite rates count as the largest numbers of f32."""
    s = Scan([(count, 1, False)], 40, n, "f32", seed=n, softplus=False, bias=False)
    s.a[3], s.a[5] = -np.inf, np.inf
    s.dt[:] = 0.0
    a = s.upload()
    a.max_new = count
    run(a)
    assert np.array_equal(s.d_state.get().reshape(s.state.shape), s.state)


@pytest.mark.parametrize("n", [5, 16, 40])
@pytest.mark.parametrize("kind", ["nothing", "little"])
def test_states_that_grow_beyond_a_stretch(n, kind):
    """d below 0 (softplus off): a factor of more than f32 holds lies between the ends of two stretches; the states that it meets are zeros, or so small that they stay in range.
    Per row 5 u of the state (an exponential 2^-22 + u, a product and an addition), the exponent's own rounding 2 u of 300 at most: 600 x 5 u + 600 u < 2^-12."""
    s = Scan([(600, 0, False)], 40, n, "f32", softplus=False, bias=False, gate=False, skip=False, seed=n)
    s.a = np.full_like(s.a, -1.0)
    s.b, s.c = np.abs(s.b), np.abs(s.c)
    s.x[:] = 0.0
    if kind == "nothing":  # e^112 in 64 rows, of zeros
        s.dt[:] = -0.25
        s.dt[:, 5:9] = -1.75
        s.state[:] = 0.0
        s.x[560:, :] = -1.0  # (d is below 0: so are the products)
    else:  # e^100 in the second 64 rows, of 1e-37
        s.dt[:] = 0.0
        s.dt[64:128] = -1.5625
        s.state[:] = 1e-37
    a = s.upload()
    run(a)
    got, want, got_state, state = same_kinds(s)
    for g, w in ((got, want), (got_state, state)):
        assert np.isfinite(w).all() and (np.abs(g - w) <= 2.0 ** -12 * np.abs(w)).all()


@pytest.mark.parametrize("kind,n,groups", [("f32", 16, 1), ("bf16", 5, 3), ("f16", 64, 2)])
@pytest.mark.parametrize("max_new", [0, 640])
def test_single_rows_beside_prompts_in_stretches(kind, n, groups, max_new):
    """As a server's step has them: single rows and prompts in any order, rows between them that nobody has, prompts that begin anywhere in a stretch and are a row longer or shorter than one."""
    counts = [1, 640, 1, 1, 129, 1, 0, 128, 127, 1, 257, 1, 1, 64, 65, 1, 63]
    rng = np.random.default_rng(n)
    order = rng.permutation(len(counts))
    first, at = np.zeros(len(counts), int), 3
    for i in order:
        first[i] = at
        at += counts[i] + int(rng.integers(0, 3))
    slots = rng.permutation(len(counts) + 2)[:len(counts)]
    info = np.array([first, counts, slots, rng.integers(0, 2, len(counts))], np.int32)
    s = Scan(info, 60, n, kind, groups=groups, seed=n, slow=True, slots=len(counts) + 2, tokens=at + 5)
    a = s.upload()
    a.max_new = max_new
    ws = run(a)
    assert ws.numel() > 16
    s.verify(max_new)


@pytest.mark.parametrize("n", [5, 16, 40])
def test_infinite_states_that_fade_over_a_stretch(n):
    """A factor of e^-5 a row: an infinite state stays so, however many rows there are, and a finite one leaves nothing behind."""
    s = Scan([(300, 1, False)], 40, n, "f32", bias=False, gate=False, skip=False, seed=n)
    s.dt[:], s.a[:] = 5.0, -1.0
    s.b, s.c = np.abs(s.b) + 0.125, np.abs(s.c) + 0.125
    s.state[1, 3], s.state[1, 4], s.state[1, 5] = np.inf, -np.inf, 3e38
    run(s.upload())
    got, want, got_state, state = same_kinds(s)
    there = np.isfinite(want)
    assert there[:, 5].all() and np.allclose(got[there], want[there], rtol=1e-4, atol=1e-4) and np.allclose(got_state[1, 5], state[1, 5], rtol=1e-4, atol=1e-4)
