"""Whether what a selection returned is right, successor by successor (include/b200_state.h): each pair of beam and token is one that there is, appears once, has the score that it is given, in its
place; the slot is its beam's."""
import numpy as np

# A score is off by what the normaliser is: a sum of exponentials of 2^-22 each, whose arguments' roundings count where the exponentials do (2^-24), and by 64-bit sums.  2^-21 is more than both.
SCORE = 2.0 ** -21


def successors(logits, score, ended, n_beams, end_token):
    """Scores in 64 bits of all successors, [requests, beams * vocab], -inf where there is none."""
    rows, v = logits.shape
    out = np.full((rows, v), -np.inf)
    for i in range(rows):
        s = float(score[i])
        if not s > -np.inf:
            continue
        if ended is not None and ended[i]:
            out[i, end_token] = s
            continue
        x = np.where(np.isnan(logits[i]), -np.inf, logits[i])
        m = x.max()
        if m == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            out[i] = np.where(x == np.inf, s - np.log((x == np.inf).sum()), -np.inf) if m == np.inf else s + ((x - m) - np.log(np.exp(x - m).sum()))
    return out.reshape(rows // n_beams, n_beams * v)


def faults(logits, score, ended, slot, n_beams, keep, end_token, to_score, to_beam, to_token, to_slot):
    """What is wrong with the results, [requests, keep] each, as a list of texts."""
    v, all_scores, bad = logits.shape[1], successors(logits, score, ended, n_beams, end_token), []
    for r, p in enumerate(all_scores):
        n = min(keep, int((p > -np.inf).sum()))
        best = np.sort(p)[::-1][:n]
        seen = set()
        for k in range(keep):
            b, t, s = int(to_beam[r, k]), int(to_token[r, k]), float(to_score[r, k])
            at = f"request {r}, place {k}: "
            if k >= n:
                if (b, t, s) != (-1, -1, -np.inf) or (to_slot is not None and to_slot[r, k] != -1):
                    bad.append(at + f"({b}, {t}, {s}) where nothing is left")
                continue
            if not (0 <= b < n_beams and 0 <= t < v):
                bad.append(at + f"no such successor ({b}, {t})")
                continue
            mine = p[b * v + t]
            if (b, t) in seen:
                bad.append(at + f"({b}, {t}) a second time")
            seen.add((b, t))
            if mine == -np.inf:
                bad.append(at + f"({b}, {t}) is no successor")
                continue
            if not abs(s - mine) <= SCORE + abs(mine) * 2.0 ** -24:
                bad.append(at + f"({b}, {t}) has score {mine}, not {s}")
            if not mine >= best[k] - 2 * SCORE:  # (two beams' normalisers)
                bad.append(at + f"({b}, {t}) of score {mine}, where {best[k]} belongs")
            if to_slot is not None and to_slot[r, k] != slot[r * n_beams + b]:
                bad.append(at + f"slot {to_slot[r, k]}, not beam {b}'s")
            if k and (to_beam[r, k - 1], to_score[r, k - 1]) == (b, s) and logits[r * n_beams + b, to_token[r, k - 1]] == logits[r * n_beams + b, t] and to_token[r, k - 1] > t:
                bad.append(at + f"equal tokens {to_token[r, k - 1]} and {t} of a beam the wrong way round")
    return bad
