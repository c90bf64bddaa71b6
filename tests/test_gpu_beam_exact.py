"""Selections on the GPU, looked at one successor at a time: each that is returned is a successor, with the score that it has, in its place; and it is the same whenever it is made."""
import ctypes as C

import numpy as np
import pytest
import torch

import beam_check
from koboldcpp_b200.lib import check, lib
from test_gpu_beam import Select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,beams,vocab,keep", [(64, 1, 1, 1), (64, 2, 3, 5), (40, 4, 40, 8), (16, 8, 600, 16), (8, 16, 1300, 64)])
def test_few_candidates_again_and_again(requests, beams, vocab, keep):
    """Lists so short that some warps are through them before others have begun: hundreds of calls, all with the first one's results."""
    s = Select(requests, beams, vocab, keep, seed=vocab)
    s.run().verify()
    first = [t.clone() for t in s.to]
    for _ in range(300):
        for t in s.to:
            t.fill_(77)
        check(lib().b200_op_beam_select(C.byref(s.args), s.ws.data_ptr(), s.ws.numel(), None))
        assert all(torch.equal(a, b) for a, b in zip(s.to, first))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [40, 2000, 70000])
def test_scores_and_logits_of_plus_infinity(kind, vocab):
    """A beam of score +inf comes before all others; where its row has logits of +inf, these are its only successors."""
    s = Select(3, 4, vocab, 12, kind, seed=vocab)
    s.score[[1, 6]] = np.inf
    s.logits[1, [3, 30, vocab - 1]] = np.inf
    s.logits[2, 5] = np.inf
    s.run()
    beam, token, score, slot = (s.to[i][:-1].cpu().numpy().reshape(3, 12) for i in (1, 2, 0, 3))
    assert beam[0, :4].tolist() == [1, 1, 1, 2] and token[0, :4].tolist() == [3, 30, vocab - 1, 5] and (score[0, :3] == np.inf).all()
    assert score[0, 3] == s.score[2] and (np.diff(score[0, 3:]) <= 0).all() and (beam[0, 4:] % 3 == 0).all()
    assert (beam[1] == 2).all() and token[1].tolist() == list(range(12)) and (score[1] == np.inf).all()  # (equal ones by their place)
    assert np.isfinite(score[2]).all() and np.array_equal(slot, np.take_along_axis(s.slot.reshape(3, 4), beam, 1))


def faults(s):
    r, b, _ = s.shape
    got = [t[:-1].cpu().numpy().reshape(r, s.keep) for t in s.to]
    return beam_check.faults(s.logits, s.score, s.ended, s.slot, b, s.keep, s.end, *got[:3], got[3] if s.slot is not None else None)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("requests,beams,vocab,keep", [(1, 1, 1, 1), (1, 1, 7, 3), (2, 4, 100, 8), (3, 5, 511, 5), (1, 8, 513, 16), (2, 3, 4097, 6), (1, 64, 1025, 128), (5, 4, 32003, 8), (1, 2, 200001, 4),
                                                       (2, 32, 70000, 64), (3, 16, 9000, 128), (7, 7, 777, 7)])
def test_every_successor(kind, requests, beams, vocab, keep):
    for seed in range(3):
        assert faults(Select(requests, beams, vocab, keep, kind, seed=vocab + seed, ended=0.2 if beams > 2 else 0.0, gap=seed, shift=seed).run()) == []


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_every_successor_of_beams_that_are_alike(kind):
    """Beams a little apart, as those of one request are: the last places are close calls."""
    for seed in range(6):
        s = Select(4, 8, 5003, 16, kind, seed=seed)
        s.score[:] = -3.0 + np.random.default_rng(seed).normal(size=32).astype(np.float32) * 1e-4
        s.logits[:] = np.repeat(s.logits[::8], 8, axis=0)
        assert faults(s.run()) == []


def test_every_successor_where_little_is_allowed():
    for kept in (1, 3, 40):
        s = Select(3, 4, 3000, 20, "f16", seed=kept)
        allowed = np.random.default_rng(kept).choice(3000, kept, replace=False)
        mask = np.ones(3000, bool)
        mask[allowed] = False
        s.logits[:, mask] = -np.inf
        s.logits[5], s.score[8:11] = np.nan, -np.inf
        assert faults(s.run()) == []
