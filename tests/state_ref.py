"""What include/b200_state.h says, in numpy and 64 bits, each with how far f32 arithmetic may be from it.

Errors are followed to first order, in units of u = 2^-24 (half a step of f32, relative).  `ex`: what an exponential is off by, relative: the special function unit's 2^-22,
and its argument's own rounding, which counts with the argument's size.
"""
import numpy as np

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a type, relative
LEAST = {"f32": 2.0 ** -140, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half a step of the smallest numbers


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-x))


def exp_error(x):
    return 2.0 ** -22 + 3 * U * np.abs(x)


def silu_error(x):
    """Of x sigmoid(x), relative: the exponential, where it counts in 1 + e^-x, an addition, a division (2^-22) and a product."""
    return exp_error(x) + 2.0 ** -22 + 3 * U


def stored(y, tol, kind):
    """The tolerance of y once it has been rounded to its type."""
    return tol + (np.abs(y) + tol) * HALF[kind] + LEAST[kind]


def sequences(info, n_slots, n_tokens, max_new=0):
    """(first, count, slot, begins) of each sequence as far as it can be."""
    for first, count, slot, begins in np.asarray(info).T.tolist():
        if first < 0 or first >= n_tokens or slot < 0 or slot >= n_slots or count <= 0:
            continue
        yield first, min(count, n_tokens - first, max_new or n_tokens), slot, bool(begins)


def conv(x, w, bias, info, tail, silu, dst, kind, max_new=0):
    """dst and tail [slots, taps - 1, channels] behind the call, and dst's tolerance."""
    taps = w.shape[1]
    dst, tail, tol = dst.copy(), tail.copy(), np.zeros_like(dst)
    for first, count, slot, begins in sequences(info, tail.shape[0], x.shape[0], max_new):
        u = np.concatenate([np.zeros_like(tail[slot]) if begins else tail[slot], x[first:first + count]])
        parts = [u[j:j + count] * w[:, j] for j in range(taps)]
        y = sum(parts) + (0 if bias is None else bias)
        e = (taps + 1) * U * (sum(np.abs(p) for p in parts) + (0 if bias is None else np.abs(bias)))
        if silu:
            e = 1.1 * e + np.abs(y * sigmoid(y)) * silu_error(y)  # (the derivative of silu is below 1.1)
            y = y * sigmoid(y)
        dst[first:first + count], tol[first:first + count] = y, stored(y, e, kind)
        if taps > 1:
            tail[slot] = u[count:]
    return dst, tail, tol


def scan(x, dt, b, c, z, a, dt_bias, skip, info, state, softplus, dst, kind, groups=1, max_new=0):
    """dst and state [slots, channels, d_state] behind the call, and the tolerances of both.  The sum of d over a stretch of rows, where stretches meet, is off by as many roundings
    as it has terms: per row d |a| times u times the number of rows, in the exponent."""
    ch, n = a.shape
    of = np.arange(ch) // (ch // groups)
    dst, state = dst.copy(), state.copy()
    tol, state_tol = np.zeros_like(dst), np.zeros_like(state)
    for first, count, slot, begins in sequences(info, state.shape[0], x.shape[0], max_new):
        h = np.zeros_like(state[slot]) if begins else state[slot].copy()
        e, lost = np.zeros_like(h), np.zeros(h.shape, bool)
        for t in range(first, first + count):
            raw = dt[t] + (0 if dt_bias is None else dt_bias)
            raw_error = 0 if dt_bias is None else U * np.abs(raw)
            d, d_error = raw, raw_error
            if softplus:  # an exponential, and a logarithm that is off by 4 u of itself
                d = np.logaddexp(0, raw)
                d_error = raw_error + d * (exp_error(np.minimum(np.abs(raw), 30)) + 4 * U)
            turn = d[:, None] * a
            decay = np.exp(turn)
            off = exp_error(turn) + np.abs(a) * d_error[:, None] if softplus or dt_bias is not None else exp_error(turn)
            off = off + np.abs(turn) * U * count
            bt, ct = b[t].reshape(groups, n)[of], c[t].reshape(groups, n)[of]
            add = (d * x[t])[:, None] * bt
            add_error = np.abs(add) * 3 * U + np.abs(x[t][:, None] * bt) * (d_error if np.ndim(d_error) else np.full(ch, d_error))[:, None]
            e = np.where(lost, np.inf, decay * np.where(lost, 0, e) + np.abs(decay * h) * off + add_error)
            h = decay * h + add
            lost |= np.abs(h) > 2.0 ** 120  # f32 ends here, or in the products that it enters: from then on nothing is said of this state
            h = np.where(lost, 0, h)
            e = np.where(lost, np.inf, e + np.abs(h) * 2 * U)
            y = (ct * h).sum(1)
            y_error = (np.where(lost, np.inf, np.abs(ct) * np.where(lost, 0, e))).sum(1) + (np.abs(ct * h)).sum(1) * (n + 1) * U
            if skip is not None:
                y, y_error = y + skip * x[t], y_error + 2 * U * (np.abs(skip * x[t]) + np.abs(y))
            if z is not None:
                g = z[t] * sigmoid(z[t])
                y_error = np.where(lost.any(1), np.inf, np.abs(g) * np.where(lost.any(1), 0, y_error)) + np.abs(y * g) * (silu_error(z[t]) + U)
                y = y * g
            dst[t], tol[t] = y, stored(y, y_error, kind)
        state[slot], state_tol[slot] = h, e + 2.0 ** -120
    return dst, state, tol, state_tol


def select(logits, score, ended, slot, n_beams, keep, end_token):
    """Scores (64 bits), beams, tokens and slots of every request's best, [requests, keep] each."""
    rows, v = logits.shape
    out = []
    for r in range(rows // n_beams):
        found = []
        for b in range(n_beams):
            i = r * n_beams + b
            s = float(score[i])
            if not s > -np.inf:
                continue
            if ended is not None and ended[i]:
                found.append((s, b, end_token))
                continue
            x = np.where(np.isnan(logits[i]), -np.inf, logits[i])
            m = x.max()
            if m == -np.inf:
                continue
            if m == np.inf:
                p = np.where(x == np.inf, -np.log((x == np.inf).sum()), -np.inf)
            else:
                p = (x - m) - np.log(np.exp(x - m).sum())
            with np.errstate(invalid="ignore"):
                p = s + p
            best = np.lexsort((np.arange(v), -p))[:keep]
            found += [(p[t], b, int(t)) for t in best if p[t] > -np.inf]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        found = found[:keep]
        n = len(found)
        out.append(([f[0] for f in found] + [-np.inf] * (keep - n), [f[1] for f in found] + [-1] * (keep - n), [f[2] for f in found] + [-1] * (keep - n),
                    [int(slot[r * n_beams + f[1]]) for f in found] + [-1] * (keep - n) if slot is not None else None))
    return tuple(np.array([o[k] for o in out]) if out and out[0][k] is not None else None for k in range(4))


def reorder(states, src, dst, n_slots):
    """The states behind the call, and how many entries were refused."""
    refused, taken, moves = 0, set(), []
    for s, d in zip(src, dst):
        if not (0 <= s < n_slots and 0 <= d < n_slots) or d in taken:
            refused += 1
            continue
        taken.add(d)
        moves.append((s, d))
    out = []
    for x in states:
        y = x.copy()
        for s, d in moves:
            y[d] = x[s]
        out.append(y)
    return out, refused
