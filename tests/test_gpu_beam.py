"""Beam search on the GPU against tests/state_ref.py (include/b200_state.h): the selection, the reordering of slots, and a small model of recurrent layers that is searched with both."""
import ctypes as C

import numpy as np
import pytest
import torch

import koboldcpp_b200.lib as L
import state_ref as R
from koboldcpp_b200.lib import BeamSelectArgs, SlotState, SsmConvArgs, SsmScanArgs, check, lib

pytestmark = pytest.mark.gpu

TYPES = {"f32": (L.F32, torch.float32), "f16": (L.F16, torch.float16), "bf16": (L.BF16, torch.bfloat16)}


class Select:
    def __init__(self, requests, beams, vocab, keep, kind="f32", seed=0, shift=0, gap=0, ended=0.0, slots=True):
        rng = np.random.default_rng(seed)
        self.shape, self.kind, self.keep = (requests, beams, vocab), kind, keep
        rows = requests * beams
        self.logits = torch.from_numpy(rng.normal(size=(rows, vocab)).astype(np.float32) * 3).to(TYPES[kind][1]).double().numpy()
        self.score = (-10 * rng.random(rows)).astype(np.float32)
        self.ended = (rng.random(rows) < ended).astype(np.int32) if ended else None
        self.slot = rng.permutation(rows).astype(np.int32) if slots else None
        self.end, self.shift, self.gap = vocab // 2, shift, gap

    def run(self, stream=None):
        r, b, v = self.shape
        rows, t = r * b, TYPES[self.kind][1]
        flat = torch.full((self.shift + rows * (v + self.gap) + 8,), float("inf"), dtype=t, device="cuda")
        self.view = flat[self.shift:self.shift + rows * (v + self.gap)].view(rows, v + self.gap)
        self.view[:, :v] = torch.from_numpy(self.logits).to(t).cuda()
        dev = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
        self.d = [dev(self.score), dev(self.ended), dev(self.slot)]
        n = r * self.keep
        self.to = [torch.full((n + 1,), 77, dtype=torch.float32 if i == 0 else torch.int32, device="cuda") for i in range(4)]
        p = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        self.args = BeamSelectArgs(logits=self.view.data_ptr(), logits_stride=v + self.gap, score=p(self.d[0]), ended=p(self.d[1]), slot=p(self.d[2]), to_score=p(self.to[0]), to_beam=p(self.to[1]),
                                   to_token=p(self.to[2]), to_slot=p(self.to[3]) if self.slot is not None else None, n_requests=r, n_beams=b, n_vocab=v, n_keep=self.keep, end_token=self.end,
                                   type=TYPES[self.kind][0])
        size = lib().b200_beam_select_workspace_bytes(C.byref(self.args))
        self.ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
        check(lib().b200_op_beam_select(C.byref(self.args), self.ws.data_ptr(), size, stream))
        return self

    def verify(self):
        r, b, v = self.shape
        score, beam, token, slot = R.select(self.logits, self.score, self.ended, self.slot, b, self.keep, self.end)
        got = [t[:-1].cpu().numpy().reshape(r, self.keep) for t in self.to]
        assert all(t[-1].item() == 77 for t in self.to)
        # the result is a sum of f32 exponentials (2^-22 each) in 64 bits, rounded once
        there = np.isfinite(score)
        assert np.array_equal(there, np.isfinite(got[0]))
        assert (np.abs(got[0][there] - score[there]) <= 2.0 ** -21 + np.abs(score[there]) * 2.0 ** -24).all()
        same = (got[1] == beam) & (got[2] == token)
        if not same.all():  # two beams' successors that are as good as each other within the sums' error
            for i, k in np.argwhere(~same):
                near = [j for j in range(self.keep) if got[1][i, k] == beam[i, j] and got[2][i, k] == token[i, j]]
                at = score[i, near[0]] if near else score[i, -1]
                assert abs(at - score[i, k]) <= 2.0 ** -20, (i, k)
        elif slot is not None:
            assert np.array_equal(got[3], slot)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("requests,beams,vocab,keep", [(1, 1, 1, 1), (1, 1, 7, 3), (2, 4, 100, 8), (3, 5, 511, 5), (1, 8, 513, 16), (2, 3, 4097, 6), (1, 64, 1025, 128), (5, 4, 32003, 8), (1, 2, 200001, 4), (2, 32, 70000, 64)])
def test_selection(kind, requests, beams, vocab, keep):
    Select(requests, beams, vocab, keep, kind, seed=vocab, ended=0.2 if beams > 2 else 0.0).run().verify()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shift,gap", [(0, 3), (1, 0), (1, 5), (2, 2), (4, 4), (8, 7), (0, 8)])
def test_rows_at_any_place(kind, shift, gap):
    Select(2, 4, 1500, 6, kind, shift=shift, gap=gap, slots=False).run().verify()


def test_more_to_keep_than_there_is():
    s = Select(3, 2, 5, 128, ended=0.0)
    s.logits[0, 1:] = -np.inf
    s.logits[3] = -np.inf
    s.score[4:] = -np.inf
    s.run().verify()
    assert s.to[1][:11].tolist() == [x for x in s.to[1][:11].tolist() if x >= -1]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gap", [0, 1])
def test_equal_scores_go_by_their_place(kind, gap):
    """Rows of one value; rows that are equal, beam by beam, wherever they lie; more equal ones than any list holds."""
    s = Select(2, 4, 3001, 20, kind, gap=gap)
    s.logits[:4] = 0.5
    s.score[:4] = -1.0
    s.logits[4:] = s.logits[4]
    s.score[4:] = -2.0
    s.run()
    assert s.to[1][:20].tolist() == [0] * 20 and s.to[2][:20].tolist() == list(range(20))
    order = np.lexsort((np.arange(3001), -s.logits[4]))
    want, last = [], None
    for t in order[:20]:
        for t2 in [t] if last is None or s.logits[4, t] != last else []:
            same = [u for u in order[:60] if s.logits[4, u] == s.logits[4, t2]]
            want += [(b, int(u)) for b in range(4) for u in same]
            last = s.logits[4, t2]
    assert list(zip(s.to[1][20:40].tolist(), s.to[2][20:40].tolist())) == want[:20]


def test_the_same_value_for_all_tokens_of_many_beams():
    for vocab, beams, keep in ((40000, 32, 64), (600, 64, 128), (131072, 2, 128)):
        s = Select(1, beams, vocab, keep, "bf16")
        s.logits[:] = -3.0
        s.score[:] = -1.0
        s.score[0] = -5.0
        s.run()
        assert s.to[1][:keep].tolist() == [1] * keep and s.to[2][:keep].tolist() == list(range(keep))


def test_logits_that_are_masked_infinite_or_not_a_number():
    for kind, least in (("f32", float(np.finfo(np.float32).min)), ("f16", -65504.0), ("bf16", -3.3895313892515355e38)):
        s = Select(9, 2, 2000, 7, kind)
        s.logits[0, ::3] = -np.inf
        s.logits[1, 5:] = least
        s.logits[2] = least
        s.logits[3] = -np.inf
        s.logits[4, 100] = np.inf
        s.logits[5, [7, 1900, 40]] = np.inf
        s.logits[6, ::2] = np.nan
        s.logits[7] = np.nan
        s.logits[8, 1500] = -least
        s.logits[9] = -least
        s.logits[10, :1999] = -np.inf
        s.score[12] = np.nan
        s.score[14:16] = -np.inf
        s.score[16] = -1e30
        s.run().verify()


def test_a_search_that_begins():
    """All beams hold the same; one of them counts."""
    s = Select(4, 6, 5000, 6)
    s.logits[:] = np.repeat(s.logits[::6], 6, axis=0)
    s.score[:] = -np.inf
    s.score[::6] = 0.0
    s.run().verify()
    assert s.to[1][:-1].tolist() == [0] * 24


def test_all_beams_have_ended():
    s = Select(2, 4, 300, 4, ended=1.1)
    s.score[:] = [-3, -1, -2, -1, -4, -np.inf, -4, -5]
    s.run().verify()
    assert s.to[1][:-1].tolist() == [1, 3, 2, 0, 0, 2, 3, -1] and s.to[2][:-1].tolist() == [150] * 7 + [-1]


# ------------------------------------------------------------------------------------------------ reordering
def states_of(rng, slots, shapes, shift=0, gap=0):
    """Matrices [slots, words] in larger allocations, and what they hold."""
    out = []
    for n in shapes:
        flat = torch.from_numpy(rng.integers(-2**31, 2**31, size=shift + slots * (n + gap) + 4).astype(np.int32)).cuda()
        out.append((flat, flat[shift:shift + slots * (n + gap)].view(slots, n + gap)))
    return out


def move(states, shapes, src, dst, slots, stream=None):
    s = (SlotState * max(1, len(shapes)))(*[SlotState(v.data_ptr(), 4 * v.shape[1], 4 * n) for (_, v), n in zip(states, shapes)])
    ids = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (src, dst)]
    refused = torch.full((1,), 5, dtype=torch.int32, device="cuda")
    check(lib().b200_op_state_reorder(s, len(shapes), ids[0].data_ptr(), ids[1].data_ptr(), len(src), slots, refused.data_ptr(), stream))
    torch.cuda.synchronize()
    return refused.item() - 5


@pytest.mark.parametrize("slots,n", [(1, 1), (4, 4), (9, 8), (130, 128), (700, 700), (1500, 1024), (4096, 5)])
@pytest.mark.parametrize("shapes,shift,gap", [([4096, 12], 0, 0), ([4, 1000, 513 * 4], 0, 4), ([1, 7, 333], 0, 0), ([100], 1, 3)])
def test_reordering(slots, n, shapes, shift, gap):
    rng = np.random.default_rng(slots + n)
    states = states_of(rng, slots, shapes, shift, gap)
    before = [f.cpu().numpy().copy() for f, _ in states]
    dst = rng.permutation(slots)[:n]
    for kind in range(3):
        src = rng.permutation(dst) if kind == 0 else np.roll(dst, 1) if kind == 1 else rng.choice(slots, n)
        held = [v[:, :m].cpu().numpy() for (_, v), m in zip(states, shapes)]
        assert move(states, shapes, src.tolist(), dst.tolist(), slots) == 0
        want, _ = R.reorder(held, src.tolist(), dst.tolist(), slots)
        for (flat, v), m, w in zip(states, shapes, want):
            assert np.array_equal(v[:, :m].cpu().numpy(), w)
    for (flat, v), m, b in zip(states, shapes, before):  # what lies between the slots' bytes
        now = flat.cpu().numpy()
        here = np.ones(now.shape, bool)
        here[shift:shift + v.numel()] = (np.arange(v.shape[1]) >= m)[None].repeat(slots, 0).reshape(-1)
        assert np.array_equal(now[here], b[here])


def test_moves_that_cannot_be():
    rng = np.random.default_rng(1)
    states, shapes = states_of(rng, 6, [40, 8]), [40, 8]
    held = [v.cpu().numpy() for _, v in states]
    src, dst = [0, 6, 1, -1, 2, 3, 4, 2**31 - 1], [1, 2, 1, 3, -2**31, 2, 2, 5]
    want, refused = R.reorder(held, src, dst, 6)
    assert move(states, shapes, src, dst, 6) == refused == 6
    for (_, v), w in zip(states, want):
        assert np.array_equal(v.cpu().numpy(), w)
    assert move([], [], [0, 9], [1, 1], 4) == 1
    assert move(states, shapes, [0, 1], [0, 1], 6) == 0


def test_more_states_than_a_launch_takes():
    rng = np.random.default_rng(2)
    shapes = [8 + 4 * (i % 5) for i in range(300)]
    states = states_of(rng, 5, shapes)
    held = [v.cpu().numpy() for _, v in states]
    want, _ = R.reorder(held, [1, 2, 0, 7], [0, 1, 2, 3], 5)
    assert move(states, shapes, [1, 2, 0, 7], [0, 1, 2, 3], 5) == 1
    for (_, v), w in zip(states, want):
        assert np.array_equal(v.cpu().numpy(), w)


# ------------------------------------------------------------------------------------------------ together
def test_a_recurrent_model_searched_with_beams():
    """Embedding, two layers of convolution and scan, a head: prompts of two requests, then steps that select, reorder the slots of all layers and go on, the whole step captured once and
    replayed.  Beside it the same search in numpy and 64 bits, every beam with its own copy of its history."""
    rng = np.random.default_rng(11)
    width, n, taps, vocab, layers, requests, beams, steps, end = 64, 16, 4, 600, 2, 2, 3, 6, 5
    f = lambda *s, std=1.0: (rng.normal(size=s) * std).astype(np.float32)  # noqa: E731
    embed, head = f(vocab, width), f(width, vocab, std=2.0 / np.sqrt(width))
    head[:, end] += 0.25
    w = [dict(conv=f(width, taps, std=0.5), bias=f(width, std=0.1), bc=f(width, 2 * n, std=1 / 8), dt=f(width, width, std=1 / 8), a=-np.exp(f(width, n, std=0.5)).astype(np.float32),
              dt_bias=f(width, std=0.3), skip=f(width)) for _ in range(layers)]
    prompts = [rng.integers(0, vocab, size=k).tolist() for k in (19, 7)]

    # ---- in 64 bits: a model step for one sequence
    def forward64(tokens, mem):
        x = embed[tokens].astype(np.float64)
        out = []
        for k, p in enumerate(w):
            tail, state = mem[k] if mem else (np.zeros((1, taps - 1, width)), np.zeros((1, width, n)))
            info = [[0], [len(tokens)], [0], [0]]
            u, tail, _ = R.conv(x, p["conv"].astype(np.float64), p["bias"].astype(np.float64), info, tail, True, np.zeros_like(x), "f32")
            bc = u @ p["bc"]
            y, state, _, _ = R.scan(u, u @ p["dt"], bc[:, :n], bc[:, n:], x, p["a"].astype(np.float64), p["dt_bias"].astype(np.float64), p["skip"].astype(np.float64), info, state, True,
                                    np.zeros_like(x), "f32")
            x = x + y
            out.append((tail, state))
        return x[-1] @ head, out

    # ---- on the device
    rows = requests * beams
    dev = lambda a, t=torch.float32: torch.from_numpy(np.ascontiguousarray(a)).to(t).cuda()  # noqa: E731
    d_embed, d_head = dev(embed), dev(head)
    dw = [{k: dev(v) for k, v in p.items()} for p in w]
    slots = dev(rng.permutation(rows + 2)[:rows], torch.int32)
    tails, states = (torch.full((layers, rows + 2, m), float("nan"), device="cuda") for m in ((taps - 1) * width, width * n))
    each = (SlotState * (2 * layers))(*[SlotState(s.data_ptr(), 4 * s.shape[1], 4 * s.shape[1]) for m in (tails, states) for s in m])
    room = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")

    def forward(x, info, longest, stream):
        t = x.shape[0]
        for k, p in enumerate(dw):
            u, y = torch.empty_like(x), torch.empty_like(x)
            a = SsmConvArgs(x=x.data_ptr(), x_stride=width, w=p["conv"].data_ptr(), bias=p["bias"].data_ptr(), seq_info=info.data_ptr(), tail=tails[k].data_ptr(), slot_stride=tails.shape[2],
                            dst=u.data_ptr(), dst_stride=width, n_seq=info.shape[1], n_slots=rows + 2, n_tokens=t, max_new=longest, channels=width, taps=taps, silu=1, type=L.F32)
            check(lib().b200_op_ssm_conv(C.byref(a), stream))
            bc, dt = u @ p["bc"], u @ p["dt"]
            a = SsmScanArgs(x=u.data_ptr(), dt=dt.data_ptr(), x_stride=width, dt_stride=width, b=bc.data_ptr(), c=bc.data_ptr() + 4 * n, b_stride=2 * n, c_stride=2 * n, z=x.data_ptr(), z_stride=width,
                            a=p["a"].data_ptr(), dt_bias=p["dt_bias"].data_ptr(), d=p["skip"].data_ptr(), seq_info=info.data_ptr(), state=states[k].data_ptr(), slot_stride=states.shape[2],
                            dst=y.data_ptr(), dst_stride=width, n_seq=info.shape[1], n_slots=rows + 2, n_tokens=t, max_new=longest, channels=width, d_state=n, groups=1, softplus=1, type=L.F32)
            check(lib().b200_op_ssm_scan(C.byref(a), room.data_ptr(), room.numel(), stream))
            x = x + y
        return x

    score, ended = torch.full((rows,), -float("inf"), device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    score[::beams] = 0.0
    logits = torch.zeros(rows, vocab, device="cuda")
    to = [torch.zeros(rows, dtype=torch.float32 if i == 0 else torch.int32, device="cuda") for i in range(4)]
    sel = BeamSelectArgs(logits=logits.data_ptr(), logits_stride=vocab, score=score.data_ptr(), ended=ended.data_ptr(), slot=slots.data_ptr(), to_score=to[0].data_ptr(), to_beam=to[1].data_ptr(),
                         to_token=to[2].data_ptr(), to_slot=to[3].data_ptr(), n_requests=requests, n_beams=beams, n_vocab=vocab, n_keep=beams, end_token=end, type=L.F32)
    sel_ws = torch.empty(lib().b200_beam_select_workspace_bytes(C.byref(sel)), dtype=torch.uint8, device="cuda")
    step_info = torch.stack([torch.arange(rows, device="cuda", dtype=torch.int32), torch.ones(rows, dtype=torch.int32, device="cuda"), slots, torch.zeros(rows, dtype=torch.int32, device="cuda")]).contiguous()

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        st = stream.cuda_stream
        flat = torch.tensor(sum(prompts, []), device="cuda")
        lens = [len(p) for p in prompts]
        info = torch.tensor([[0, lens[0]], lens, slots[::beams].tolist(), [1, 1]], dtype=torch.int32, device="cuda")
        x = forward(d_embed[flat], info, max(lens), st)
        last = torch.tensor([lens[0] - 1, sum(lens) - 1], device="cuda")
        logits.copy_((x[last] @ d_head).repeat_interleave(beams, 0))

        def step():
            check(lib().b200_op_beam_select(C.byref(sel), sel_ws.data_ptr(), sel_ws.numel(), st))
            check(lib().b200_op_state_reorder(each, len(each), to[3].data_ptr(), slots.data_ptr(), rows, rows + 2, None, st))
            parent = to[1].long() + torch.arange(rows, device="cuda") // beams * beams
            ended.copy_(((ended[parent] != 0) | (to[2] == end)).int())
            score.copy_(to[0])
            logits.copy_(forward(d_embed[to[2].long()], step_info, 1, st) @ d_head)

        found = []
        step()  # (warm)
        found.append([t.clone() for t in to])
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        g.capture_begin()
        step()
        g.capture_end()
        for _ in range(steps - 1):
            g.replay()
            found.append([t.clone() for t in to])
    torch.cuda.synchronize()

    # ---- the search in 64 bits
    for r in range(requests):
        first, mem = forward64(prompts[r], None)
        live = [(0.0, False, first, mem)] + [(-np.inf, False, first, mem)] * (beams - 1)
        for k in range(steps):
            sc, be, tk, _ = R.select(np.stack([b[2] for b in live]), np.array([b[0] for b in live]), np.array([b[1] for b in live]), None, beams, beams, end)
            got = [t[r * beams:(r + 1) * beams].cpu().numpy() for t in found[k]]
            assert got[1].tolist() == be[0].tolist() and got[2].tolist() == tk[0].tolist(), (r, k, got, sc, be, tk)
            # logits are sums of 64 products in f32 of layers whose errors are some 1e-6: far below this
            assert np.allclose(got[0], sc[0], atol=2e-3)
            live = [(s, live[b][1] or t == end, *forward64([t], live[b][3])) for s, b, t in zip(sc[0], be[0].tolist(), tk[0].tolist())]
