"""Scans in stretches, in 64 bits, as the sum over stretches that they are: h behind a stretch = exp(a * sum of d) * h before it + what the stretch makes from nothing.

The tolerances follow a row by row evaluation (as tests/state_ref.py) inside a stretch, and say apart what joining the stretches may add: the sum of d is made of f32 sums of at most 16 terms and 64-bit
ones and rounded once (20 u of itself at most), times a with its own roundings, in two exponentials."""
import numpy as np

from state_ref import U, exp_error


def softplus(raw):
    return np.logaddexp(0, raw)


SUM = 20 * U     # of the sum of d over a stretch, relative
FACTOR = 2.0 ** -21 + 3 * U  # of a stretch's factor by itself: two exponentials, two products


def carry_error(h, turn):
    """Of exp(turn) h, where turn is a times the sum of d over a stretch."""
    return np.abs(np.exp(turn) * h) * (FACTOR + np.abs(turn) * (SUM + 4 * U))


def step(h, e, d, d_error, x, b, a):
    """State and its error behind a row."""
    turn = d[:, None] * a
    decay, add = np.exp(turn), (d * x)[:, None] * b
    off = exp_error(turn) + np.abs(a) * d_error[:, None]
    e = decay * e + np.abs(decay * h) * off + np.abs(add) * 3 * U + np.abs(x[:, None] * b) * d_error[:, None]
    h = decay * h + add
    return h, e + np.abs(h) * 2 * U


def scan(x, raw, b, c, a, state, stretch, sum_of=lambda d: d.sum(0), is_softplus=True):
    """One sequence, one group.  y, the state behind the last row, and their tolerances.  sum_of: the sum of d over a stretch (tests put mistakes in here)."""
    rows, ch = x.shape
    d = softplus(raw) if is_softplus else raw
    d_error = d * (2.0 ** -22 + 1.8e-7 + 5 * U) if is_softplus else np.zeros_like(d)  # (as tests/test_gpu_ssm_precision.py has it)
    y, tol = np.zeros_like(x), np.zeros_like(x)
    start, start_error = state.copy(), np.zeros_like(state)
    for r0 in range(0, rows, stretch):
        r1 = min(rows, r0 + stretch)
        h, e = start, start_error
        end, end_error = np.zeros_like(state), np.zeros_like(state)
        for t in range(r0, r1):
            h, e = step(h, e, d[t], d_error[t], x[t], b[t], a)
            end, end_error = step(end, end_error, d[t], d_error[t], x[t], b[t], a)
            y[t] = (h * c[t]).sum(1)
            tol[t] = (np.abs(c[t]) * e).sum(1) + (np.abs(c[t] * h)).sum(1) * (a.shape[1] + 1) * U + np.abs(y[t]) * U
        if r1 == rows:
            return y, h, tol, e
        turn = sum_of(d[r0:r1])[:, None] * a
        factor = np.exp(turn)
        start_error = factor * start_error + carry_error(start, turn) + np.abs(factor * start) * np.abs(a) * d_error[r0:r1].sum(0)[:, None] + end_error
        start = factor * start + end
        start_error = start_error + np.abs(start) * U


def stretch_of(size, n_tokens, channels, d_state):
    """The rows of a stretch, from what the call asks for: a whole number of eights, of which n_tokens make so many places."""
    places = size // (4 * channels * (2 * d_state + 1))
    found = [s for s in range(64, n_tokens, 8) if -(-n_tokens // s) == places]
    assert len(found) == 1, found
    return found[0]


def fading(rows, ch, n, turn, seed):
    """Steps and rates of states that lose a factor of up to e^-turn in so many rows: steps of one size with many bits, so that each addition to a sum of f32 is rounded the same way."""
    rng = np.random.default_rng(seed)
    step_size = rng.uniform(0.05, 0.1, ch).astype(np.float32).astype(np.float64)
    a = -(turn / (rows * step_size))[:, None] * rng.uniform(0.5, 1, (ch, n))
    return step_size, a.astype(np.float32).astype(np.float64)
