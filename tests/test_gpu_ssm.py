"""Short convolutions and selective state space scans on the GPU against tests/state_ref.py (include/b200_state.h), whose tolerances follow every rounding of a row by row evaluation."""
import ctypes as C

import numpy as np
import pytest
import torch

import koboldcpp_b200.lib as L
import state_ref as R
from koboldcpp_b200.lib import SsmConvArgs, SsmScanArgs, check, lib

pytestmark = pytest.mark.gpu

TYPES = {"f32": (L.F32, torch.float32), "f16": (L.F16, torch.float16), "bf16": (L.BF16, torch.bfloat16)}


def rounded(a, kind):
    """a as the type holds it, in 64 bits."""
    return torch.from_numpy(np.asarray(a, np.float32)).to(TYPES[kind][1]).double().numpy()


class Rows:
    """A matrix of rows on the device: `shift` values behind an allocation's start, `gap` values between rows that nobody may touch."""

    def __init__(self, a, kind, shift=0, gap=0):
        t, n = TYPES[kind][1], a.shape[1]
        self.stride, self.gap = n + gap, gap
        self.all = torch.full((shift + a.shape[0] * self.stride + 16,), 7.0, dtype=t, device="cuda")
        self.view = self.all[shift:shift + a.shape[0] * self.stride].view(a.shape[0], self.stride)
        self.view[:, :n] = torch.from_numpy(np.ascontiguousarray(a)).to(t).cuda()
        self.n, self.shift = n, shift
        self.ptr = self.view.data_ptr()

    def get(self):
        assert bool((self.view[:, self.n:] == 7).all()) and bool((self.all[:self.shift] == 7).all()) and bool((self.all[-16:] == 7).all()), "values beside the rows were written"
        return self.view[:, :self.n].double().cpu().numpy()


def vec(a, dtype=torch.float32):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def info_of(seqs):
    """seqs: (count, slot, begins) one behind the other."""
    first = np.concatenate([[0], np.cumsum([s[0] for s in seqs])])[:-1]
    return np.array([first, [s[0] for s in seqs], [s[1] for s in seqs], [int(s[2]) for s in seqs]], np.int32)


def rows_of_one(info, n_slots, tokens, max_new):
    """Rows that no two sequences claim: what others hold is not said."""
    claims = np.zeros(tokens, int)
    for first, count, _, _ in R.sequences(info, n_slots, tokens, max_new):
        claims[first:first + count] += 1
    return claims < 2


def near(got, want, tol):
    assert got.shape == want.shape
    off = np.abs(got - want) > tol
    assert not off.any(), (int(off.sum()), np.argwhere(off)[:4].tolist(), float(np.max(np.abs(got - want) / np.maximum(tol, 1e-300))))


# ------------------------------------------------------------------------------------------------ convolution
class Conv:
    def __init__(self, seqs, channels, taps, kind="f32", bias=True, silu=True, slots=None, tokens=None, seed=0, shift=0, gap=0, slot_gap=0):
        rng = np.random.default_rng(seed)
        self.info = info_of(seqs) if not isinstance(seqs, np.ndarray) else seqs
        self.tokens = int(self.info[1].sum()) if tokens is None else tokens
        self.slots = int(self.info[2].max()) + 2 if slots is None else slots
        self.kind, self.taps, self.silu = kind, taps, silu
        self.x = rounded(rng.normal(size=(self.tokens, channels)), kind)
        self.w = rng.normal(size=(channels, taps)).astype(np.float32).astype(np.float64)
        self.bias = rng.normal(size=channels).astype(np.float32).astype(np.float64) if bias else None
        self.tail = rounded(rng.normal(size=(self.slots, taps - 1, channels)), kind)
        self.dst = rounded(rng.normal(size=(self.tokens, channels)), kind)
        self.shift, self.gap, self.slot_gap = shift, gap, slot_gap

    def upload(self):
        self.d_x, self.d_dst = Rows(self.x, self.kind, self.shift, self.gap), Rows(self.dst, self.kind, self.shift, self.gap)
        self.d_tail = Rows(self.tail.reshape(self.slots, -1) if self.taps > 1 else np.zeros((self.slots, 1)), "f32", gap=self.slot_gap)
        self.d_w, self.d_bias, self.d_info = vec(self.w), vec(self.bias), vec(self.info, torch.int32)
        return SsmConvArgs(x=self.d_x.ptr, x_stride=self.d_x.stride, w=ptr(self.d_w), bias=ptr(self.d_bias), seq_info=ptr(self.d_info), tail=self.d_tail.ptr, slot_stride=self.d_tail.stride,
                           dst=self.d_dst.ptr, dst_stride=self.d_dst.stride, n_seq=self.info.shape[1], n_slots=self.slots, n_tokens=self.tokens, channels=self.x.shape[1], taps=self.taps,
                           silu=int(self.silu), type=TYPES[self.kind][0])

    def verify(self, max_new=0):
        dst, tail, tol = R.conv(self.x, self.w, self.bias, self.info, self.tail, self.silu, self.dst, self.kind, max_new)
        got, mine = self.d_dst.get(), rows_of_one(self.info, self.slots, self.tokens, max_new)
        untouched = tol == 0
        assert np.array_equal(got[untouched], self.dst[untouched])
        near(got[mine], dst[mine], tol[mine])
        if self.taps > 1:
            assert np.array_equal(self.d_tail.get().reshape(tail.shape), tail)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("taps", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("channels", [1, 37, 64, 1032])
def test_convolution(kind, taps, channels):
    c = Conv([(1, 3, False), (2, 0, True), (0, 1, False), (15, 5, False), (16, 4, True), (17, 2, False), (70, 6, False)], channels, taps, kind, seed=taps)
    check(lib().b200_op_ssm_conv(C.byref(c.upload()), None))
    c.verify()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shift,gap", [(0, 8), (1, 0), (0, 3), (2, 6), (8, 24)])
def test_convolution_at_any_place(kind, shift, gap):
    for bias, silu in ((False, False), (True, False), (False, True)):
        c = Conv([(19, 1, False), (3, 0, True)], 72, 4, kind, bias, silu, shift=shift, gap=gap, slot_gap=5)
        check(lib().b200_op_ssm_conv(C.byref(c.upload()), None))
        c.verify()


def test_convolution_leaves_out_what_cannot_be():
    """Slots outside, rows outside the batch, rows that belong to nobody, sequences longer than max_new."""
    for max_new in (0, 20):
        info = np.array([[0, 5, 12, 90, 30, -3, 60, 99], [5, 4, 9, 30, 25, 4, 0, 1], [0, 9, -1, 3, 1, 2, 4, 5], [0, 0, 1, 0, 0, 0, 0, 1]], np.int32)
        c = Conv(info, 40, 4, "f32", slots=6, tokens=100)
        a = c.upload()
        a.max_new = max_new
        check(lib().b200_op_ssm_conv(C.byref(a), None))
        c.verify(max_new)


def test_convolution_of_sequences_of_one_length():
    c = Conv([(21, 0, False), (21, 1, False), (21, 2, False)], 48, 4, "f16", slots=3)
    a = c.upload()
    a.seq_info = None
    check(lib().b200_op_ssm_conv(C.byref(a), None))
    c.verify()


@pytest.mark.parametrize("taps", [4, 5])
def test_values_that_are_not_finite_stay_with_their_channel_and_taps(taps):
    c = Conv([(40, 0, False)], 24, taps, "f32")
    c.x[7, 3], c.x[9, 5], c.tail[0, 0, 8] = np.nan, np.inf, np.nan
    clean = Conv([(40, 0, False)], 24, taps, "f32")
    check(lib().b200_op_ssm_conv(C.byref(c.upload()), None))
    check(lib().b200_op_ssm_conv(C.byref(clean.upload()), None))
    got, want = c.d_dst.get(), clean.d_dst.get()
    hit = np.zeros(got.shape, bool)
    hit[7:7 + taps, 3] = hit[9:9 + taps, 5] = hit[:1, 8] = True
    assert np.isnan(got[7:7 + taps, 3]).all() and not np.isfinite(got[:1, 8]).any()
    assert np.array_equal(got[~hit], want[~hit])


def test_a_prompt_at_once_and_in_portions():
    whole = Conv([(70, 1, True)], 64, 4, "bf16")
    check(lib().b200_op_ssm_conv(C.byref(whole.upload()), None))
    parts = Conv([(70, 1, True)], 64, 4, "bf16")
    a = parts.upload()
    at = 0
    for n in (1, 2, 1, 33, 3, 30):
        info = vec(np.array([[at], [n], [1], [int(at == 0)]]), torch.int32)
        a.seq_info = info.data_ptr()
        check(lib().b200_op_ssm_conv(C.byref(a), None))
        at += n
    torch.cuda.synchronize()
    assert np.array_equal(whole.d_dst.get(), parts.d_dst.get()) and np.array_equal(whole.d_tail.get(), parts.d_tail.get())


# ------------------------------------------------------------------------------------------------ scan
class Scan:
    def __init__(self, seqs, channels, n, kind="f32", groups=1, gate=True, skip=True, bias=True, softplus=True, slots=None, tokens=None, seed=0, shift=0, gap=0, slot_gap=0, slow=False):
        rng = np.random.default_rng(seed)
        self.info = info_of(seqs) if not isinstance(seqs, np.ndarray) else seqs
        t = self.tokens = int(self.info[1].sum()) if tokens is None else tokens
        self.slots = int(self.info[2].max()) + 2 if slots is None else slots
        self.kind, self.groups, self.softplus, self.n, self.ch = kind, groups, softplus, n, channels
        f = lambda *s: rng.normal(size=s).astype(np.float32).astype(np.float64)  # noqa: E731
        self.x, self.z, self.dst = rounded(f(t, channels), kind), rounded(f(t, channels), kind) if gate else None, rounded(f(t, channels), kind)
        self.dt = rounded(f(t, channels) * 1.5 - 2 if softplus else np.abs(f(t, channels)) * 0.2, kind)
        self.b, self.c = rounded(f(t, groups * n), kind), rounded(f(t, groups * n), kind)
        self.a = -np.exp(f(channels, n) - (5 if slow else 0)).astype(np.float32).astype(np.float64)
        self.bias, self.skip = f(channels) * 0.5 if bias else None, f(channels) if skip else None
        if bias:
            self.bias = self.bias.astype(np.float32).astype(np.float64)
        self.state = f(self.slots, channels, n)
        self.shift, self.gap, self.slot_gap = shift, gap, slot_gap

    def upload(self):
        rows = lambda a: Rows(a, self.kind, self.shift, self.gap) if a is not None else None  # noqa: E731
        self.d = {k: rows(getattr(self, k)) for k in ("x", "dt", "b", "c", "z", "dst")}
        self.d_state = Rows(self.state.reshape(self.slots, -1), "f32", gap=self.slot_gap)
        self.v = {"a": vec(self.a), "dt_bias": vec(self.bias), "d": vec(self.skip), "seq_info": vec(self.info, torch.int32)}
        d = self.d
        a = SsmScanArgs(x=d["x"].ptr, dt=d["dt"].ptr, x_stride=d["x"].stride, dt_stride=d["dt"].stride, b=d["b"].ptr, c=d["c"].ptr, b_stride=d["b"].stride, c_stride=d["c"].stride,
                        z=d["z"].ptr if d["z"] else None, z_stride=d["z"].stride if d["z"] else 0, **{k: ptr(t) for k, t in self.v.items()}, state=self.d_state.ptr, slot_stride=self.d_state.stride,
                        dst=d["dst"].ptr, dst_stride=d["dst"].stride, n_seq=self.info.shape[1], n_slots=self.slots, n_tokens=self.tokens, channels=self.ch, d_state=self.n, groups=self.groups,
                        softplus=int(self.softplus), type=TYPES[self.kind][0])
        return a

    def verify(self, max_new=0, state=None):
        dst, st, tol, st_tol = R.scan(self.x, self.dt, self.b, self.c, self.z, self.a, self.bias, self.skip, self.info, self.state if state is None else state, self.softplus, self.dst, self.kind,
                                      self.groups, max_new)
        got, got_state = self.d["dst"].get(), self.d_state.get().reshape(st.shape)
        assert np.array_equal(got[tol == 0], self.dst[tol == 0])
        mine = rows_of_one(self.info, self.slots, self.tokens, max_new)
        near(got[mine], dst[mine], tol[mine])
        idle = (st_tol == 0).all((1, 2))
        assert np.array_equal(got_state[idle], self.state[idle])
        near(got_state[~idle], st[~idle], st_tol[~idle])


def run(a, stream=None, fill=0xff):
    """The call with a workspace that holds NaN before it."""
    n = lib().b200_ssm_scan_workspace_bytes(C.byref(a))
    ws = torch.full((max(n, 16),), fill, dtype=torch.uint8, device="cuda")
    if stream is not None:
        stream.wait_stream(torch.cuda.current_stream())
    check(lib().b200_op_ssm_scan(C.byref(a), ws.data_ptr(), n, stream.cuda_stream if stream is not None else None))
    return ws


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 4, 5, 8, 16, 17, 32, 33, 64, 100, 128])
def test_single_tokens(kind, n):
    s = Scan([(1, 4, False), (1, 0, True), (0, 1, False), (1, 2, False)], 70, n, kind, seed=n)
    a = s.upload()
    a.max_new = 1
    run(a)
    s.verify()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 4, 5, 8, 16, 17, 32, 33, 64, 100, 128])
@pytest.mark.parametrize("channels", [3, 64, 140])
def test_prompts(kind, n, channels):
    s = Scan([(1, 3, False), (3, 0, True), (0, 1, False), (16, 5, False), (17, 4, True), (37, 6, False)], channels, n, kind, seed=n + channels)
    run(s.upload())
    s.verify()


@pytest.mark.parametrize("groups,channels", [(2, 64), (4, 40), (8, 1040), (3, 21), (7, 7)])
@pytest.mark.parametrize("count", [1, 20])
def test_groups_of_channels(groups, channels, count):
    for n, kind in ((16, "f32"), (6, "bf16"), (64, "f16")):
        s = Scan([(count, 1, False), (count, 0, True)], channels, n, kind, groups=groups, seed=groups)
        a = s.upload()
        a.max_new = count
        run(a)
        s.verify()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shift,gap,slot_gap", [(0, 4, 0), (1, 0, 0), (0, 3, 2), (2, 6, 4), (4, 12, 1), (8, 24, 0)])
@pytest.mark.parametrize("count", [1, 18])
def test_rows_and_slots_at_any_place(kind, shift, gap, slot_gap, count):
    for gate, skip, bias, softplus in ((False, False, False, False), (True, False, True, True), (False, True, False, True), (False, False, True, False)):
        s = Scan([(count, 1, False), (count, 0, True)], 72, 16, kind, gate=gate, skip=skip, bias=bias, softplus=softplus, shift=shift, gap=gap, slot_gap=slot_gap)
        a = s.upload()
        a.max_new = count
        run(a)
        s.verify()


@pytest.mark.parametrize("kind,n,groups", [("f32", 16, 1), ("bf16", 7, 1), ("f16", 12, 2), ("bf16", 32, 1)])
def test_many_sequences_of_some_length(kind, n, groups):
    """More blocks of channels than an SM holds at once, sequences that end inside, at and behind a chunk of b and c."""
    counts = [33, 70, 64, 65, 61, 40, 66, 63] * 7
    s = Scan([(k, (i * 17) % 56, i % 5 == 0) for i, k in enumerate(counts)], 1300, n, kind, groups=groups, seed=n, gap=3)
    a = s.upload()
    a.max_new = max(counts)
    run(a)
    s.verify(a.max_new)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shift,gap,slot_gap", [(0, 4, 0), (1, 0, 0), (0, 3, 2), (2, 6, 4), (4, 12, 1), (8, 24, 0)])
def test_rows_at_any_place_in_few_longer_sequences(kind, shift, gap, slot_gap):
    for gate, skip, bias, softplus in ((False, False, False, False), (True, True, True, True)):
        s = Scan([(47, 1, False), (18, 0, True)], 72, 16, kind, gate=gate, skip=skip, bias=bias, softplus=softplus, shift=shift, gap=gap, slot_gap=slot_gap)
        a = s.upload()
        a.max_new = 47
        run(a)
        s.verify(47)


@pytest.mark.parametrize("kind,n,channels,groups", [("f32", 16, 64, 1), ("bf16", 16, 100, 1), ("f32", 5, 33, 3), ("f16", 64, 64, 2), ("f32", 128, 24, 1)])
def test_long_prompts_in_stretches(kind, n, channels, groups):
    """Few channels: sequences of several hundred rows are cut; their lengths end before, on and behind the cuts, and some have no second stretch."""
    seqs = [(640, 2, False), (1, 0, False), (639, 4, True), (31, 1, False), (32, 3, True), (33, 6, False), (0, 5, False), (257, 7, False)]
    s = Scan(seqs, channels, n, kind, groups=groups, seed=n, slow=True)
    a = s.upload()
    a.max_new = 640
    assert lib().b200_ssm_scan_workspace_bytes(C.byref(a)) > 0
    run(a)
    s.verify()


def test_states_that_hardly_fade_over_a_long_prompt():
    s = Scan([(3000, 0, False)], 40, 16, "f32", softplus=False, bias=False, seed=3, slow=True)
    s.a *= 1e-3
    s.a = s.a.astype(np.float32).astype(np.float64)
    run(s.upload())
    s.verify()


def test_scan_leaves_out_what_cannot_be():
    """Slots outside, rows outside the batch, rows that belong to nobody, sequences longer than max_new; one row a sequence, whole sequences, stretches."""
    info = np.array([[0, 5, 12, 990, 30, -3, 60, 999, 2**31 - 1], [5, 4, 9, 30, 900, 4, 0, 1, 2**31 - 1], [0, 9, -1, 3, 1, 2, 4, 5, 2], [0, 0, 1, 0, 0, 0, 0, 1, 0]], np.int32)
    for max_new in (0, 1, 20, 700):
        s = Scan(info, 40, 16, "f32", slots=6, tokens=1000, slow=True)
        a = s.upload()
        a.max_new = max_new
        run(a)
        s.verify(max_new)


@pytest.mark.parametrize("count", [1, 24, 300])
def test_states_from_elsewhere(count):
    """`from`, sequences of one length without seq_info, and a state that nobody has written yet."""
    s = Scan([(count, 0, False), (count, 1, False), (count, 2, False)], 40, 16, "f32", slots=3)
    a = s.upload()
    other = Rows(s.state.reshape(3, -1), "f32", gap=8)
    s.d_state.view[:, :] = float("nan")
    s.d_state = Rows(np.full((3, 640), np.nan), "f32", gap=4)
    a.state, a.slot_stride, a.seq_info = s.d_state.ptr, s.d_state.stride, None
    setattr(a, "from", other.ptr)
    a.from_stride = other.stride
    run(a)
    s.verify()
    assert np.array_equal(other.get(), s.state.reshape(3, -1).astype(np.float32))


@pytest.mark.parametrize("count", [1, 30, 500])
@pytest.mark.parametrize("name", ["x", "dt", "z"])
def test_results_in_place_of_an_input(count, name):
    s = Scan([(count, 1, False), (count, 0, True)], 64, 16, "bf16")
    a = s.upload()
    a.max_new = count
    run(a)
    want, state = s.d["dst"].get(), s.d_state.get()
    t = Scan([(count, 1, False), (count, 0, True)], 64, 16, "bf16")
    a = t.upload()
    a.max_new = count
    a.dst, a.dst_stride = t.d[name].ptr, t.d[name].stride
    run(a)
    assert np.array_equal(t.d[name].get(), want) and np.array_equal(t.d_state.get(), state)


@pytest.mark.parametrize("n", [16, 40])
def test_a_prompt_at_once_in_portions_and_token_by_token(n):
    """The same rows, whatever the steps: within the tolerances of both."""
    whole = Scan([(90, 1, True)], 64, n, "f32", seed=9)
    run(whole.upload())
    whole.verify()
    for portions in ([1] * 90, [40, 1, 49], [89, 1], [2] * 45):
        s = Scan([(90, 1, True)], 64, n, "f32", seed=9)
        a, at = s.upload(), 0
        for k in portions:
            info = vec(np.array([[at], [k], [1], [int(at == 0)]]), torch.int32)
            a.seq_info, a.max_new = info.data_ptr(), k
            ws = run(a)
            at += k
            torch.cuda.synchronize()
            del ws
        s.verify()


def test_exponents_at_their_ends():
    """Decays that leave nothing, states that grow, d of 0 and d that no exponential of f32 reaches."""
    s = Scan([(40, 0, False)], 32, 16, "f32", seed=5)
    s.dt[3], s.dt[4], s.dt[5, :16] = 300.0, -300.0, 90.0
    s.a[:4] = -50.0
    s.a[4:6] = 0.0
    s.a[6] = 1e-3
    run(s.upload())
    s.verify()


@pytest.mark.parametrize("count", [1, 50, 400])
def test_values_that_are_not_finite_stay_with_their_channel(count):
    """In x, dt, z: the channel's rows from there on (z: that row); in b: all channels of its group."""
    def made():
        return Scan([(count, 1, False), (count, 0, False)], 64, 16, "f32", groups=2, seed=4)
    clean, s = made(), made()
    t = count // 2
    s.x[t, 3], s.dt[t, 9], s.z[t, 40], s.state[1, 11, 2] = np.nan, np.nan, np.nan, np.inf
    s.x[count + t, 5] = np.inf
    for m in (clean, s):
        a = m.upload()
        a.max_new = count
        run(a)
    got, want = s.d["dst"].get(), clean.d["dst"].get()
    hit = np.zeros(got.shape, bool)
    hit[t:count, 3] = hit[t:count, 9] = hit[t, 40] = hit[:count, 11] = hit[count + t:, 5] = True
    assert np.isnan(got[t:count, 3]).all() and np.isnan(got[t:count, 9]).all() and np.isnan(got[t, 40]) and not np.isfinite(got[count + t:, 5]).any()
    assert np.array_equal(got[~hit], want[~hit])
    b = made()
    b.b[t, 20] = np.nan  # group 1
    a = b.upload()
    a.max_new = count
    run(a)
    got = b.d["dst"].get()
    assert np.isnan(got[t:count, 32:]).all() and np.array_equal(got[:, :32], want[:, :32]) and np.array_equal(got[count:], want[count:]) and np.array_equal(got[:t], want[:t])


def test_two_streams_and_replayed_graphs():
    """Steps of one token on a stream of their own beside prompts on another, then a captured step that is replayed: the states go on."""
    steps = Scan([(1, 0, False), (1, 1, False)], 96, 16, "f32", seed=6)
    prompt = Scan([(500, 0, True)], 48, 16, "bf16", seed=7)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    a, b = steps.upload(), prompt.upload()
    a.max_new = 1
    torch.cuda.synchronize()
    keep = [run(b, two)]
    for _ in range(3):
        keep.append(run(a, one))
    torch.cuda.synchronize()
    prompt.verify()
    state = steps.state
    for _ in range(3):
        dst, state, _, _ = R.scan(steps.x, steps.dt, steps.b, steps.c, steps.z, steps.a, steps.bias, steps.skip, steps.info, state, True, steps.dst, "f32")
    assert np.allclose(steps.d_state.get().reshape(state.shape)[:2], state[:2], rtol=1e-4, atol=1e-5)
    n = lib().b200_ssm_scan_workspace_bytes(C.byref(b))
    ws = torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(one):
        g.capture_begin()
        check(lib().b200_op_ssm_scan(C.byref(b), ws.data_ptr(), n, one.cuda_stream))
        check(lib().b200_op_ssm_scan(C.byref(a), None, 0, one.cuda_stream))
        g.capture_end()
    prompt.d["dst"].view.zero_()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    prompt.verify()  # (it begins: the slot does not matter)
    for _ in range(2):
        dst, state, _, _ = R.scan(steps.x, steps.dt, steps.b, steps.c, steps.z, steps.a, steps.bias, steps.skip, steps.info, state, True, steps.dst, "f32")
    assert np.allclose(steps.d_state.get().reshape(state.shape)[:2], state[:2], rtol=1e-4, atol=1e-5)
