"""tests/beam_check.py finds mistakes that are put into right results, wherever they are."""
import numpy as np
import pytest

import beam_check
import state_ref as R

BEAMS, KEEP, END = 3, 6, 4


def right():
    rng = np.random.default_rng(0)
    logits, score = rng.normal(size=(6, 50)) * 3, -10 * rng.random(6)
    logits[4, 3:] = -np.inf
    score[3] = -np.inf
    ended = np.array([0, 1, 0, 0, 0, 1])
    slot = rng.permutation(6)
    return dict(logits=logits, score=score, ended=ended, slot=slot), [x.copy() for x in R.select(logits, score, ended, slot, BEAMS, KEEP, END)]


def faults(inputs, found):
    s, b, t, slot = found
    return beam_check.faults(**inputs, n_beams=BEAMS, keep=KEEP, end_token=END, to_score=s.astype(np.float32), to_beam=b, to_token=t, to_slot=slot)


def test_right_results_have_none():
    inputs, found = right()
    assert found[1][1].tolist().count(-1) == 2  # (a request with fewer successors than are kept)
    assert faults(inputs, found) == []


@pytest.mark.parametrize("place", range(KEEP))
@pytest.mark.parametrize("what", ["token", "beam", "range", "twice", "score", "slot", "none"])
def test_a_mistake_at_any_place_is_found(place, what):
    inputs, found = right()
    s, b, t, slot = found
    if what == "token":
        t[0, place] = (t[0, place] + 1) % 50
    elif what == "beam":
        b[0, place] = (b[0, place] + 1) % BEAMS
        slot[0, place] = inputs["slot"][b[0, place]]
    elif what == "range":
        t[0, place] = 50
    elif what == "twice":
        for x in found:
            x[0, place] = x[0, place - 1 if place else 1]
    elif what == "score":
        s[0, place] += 2.0 ** -18
    elif what == "slot":
        slot[0, place] += 1
    else:
        for x, v in zip(found, (-np.inf, -1, -1, -1)):
            x[0, place] = v
    assert faults(inputs, found)


def test_a_result_where_nothing_is_left_is_found():
    inputs, found = right()
    found[1][1, KEEP - 1] = 0
    assert faults(inputs, found)


def test_equal_tokens_the_wrong_way_round_are_found():
    inputs, _ = right()
    inputs["logits"][0, [7, 9]] = 30.0
    found = [x.copy() for x in R.select(inputs["logits"], inputs["score"], inputs["ended"], inputs["slot"], BEAMS, KEEP, END)]
    assert faults(inputs, found) == []
    i = found[2][0].tolist().index(7)
    found[2][0, [i, i + 1]] = 9, 7
    assert faults(inputs, found)
