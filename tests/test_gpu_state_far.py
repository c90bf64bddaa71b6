"""include/b200_state.h with rows and slots further apart than 31 bits count: results are those of the same rows and slots side by side, bit by bit."""
import ctypes as C

import numpy as np
import pytest
import torch

import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import BeamSelectArgs, SlotState, SsmConvArgs, SsmScanArgs, check, lib

pytestmark = pytest.mark.gpu


def spread(a, stride):
    """The rows of a, `stride` values apart (what lies between them is whatever it is)."""
    flat = torch.empty((a.shape[0] - 1) * stride + a.shape[1], dtype=a.dtype, device="cuda")
    view = torch.as_strided(flat, a.shape, (stride, 1))
    view.copy_(a)
    return view


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("counts", [(1, 1), (7, 5)])
@pytest.mark.parametrize("n", [16, 40])
def test_scan_and_convolution(counts, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    rows, ch, taps, slots = sum(counts), 40, 4, 4
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, dt, z, bc = (r(rows, m).to(torch.bfloat16) for m in (ch, ch, ch, 2 * n))
    a, w, state, tail = -r(ch, n).abs(), r(ch, taps), r(slots, ch * n), r(slots, (taps - 1) * ch)
    info = torch.tensor([[0, counts[0]], counts, [3, 1], [0, 0]], dtype=torch.int32, device="cuda")

    def run(row, slot):
        d = {k: spread(v, row) if row else v.clone() for k, v in dict(x=x, dt=dt, z=z, bc=bc, y=torch.zeros_like(x), u=torch.zeros_like(x)).items()}
        s, t = (spread(v, slot) if slot else v.clone() for v in (state, tail))
        at, st = (lambda k: d[k].data_ptr()), (lambda k: d[k].stride(0))  # noqa: E731
        c = SsmConvArgs(x=at("x"), x_stride=st("x"), w=w.data_ptr(), seq_info=info.data_ptr(), tail=t.data_ptr(), slot_stride=t.stride(0), dst=at("u"), dst_stride=st("u"), n_seq=2, n_slots=slots,
                        n_tokens=rows, max_new=max(counts), channels=ch, taps=taps, silu=1, type=L.BF16)
        check(lib().b200_op_ssm_conv(C.byref(c), None))
        c = SsmScanArgs(x=at("u"), x_stride=st("u"), dt=at("dt"), dt_stride=st("dt"), b=at("bc"), b_stride=st("bc"), c=at("bc") + 2 * n, c_stride=st("bc"), z=at("z"), z_stride=st("z"), a=a.data_ptr(),
                        seq_info=info.data_ptr(), state=s.data_ptr(), slot_stride=s.stride(0), dst=at("y"), dst_stride=st("y"), n_seq=2, n_slots=slots, n_tokens=rows, max_new=max(counts), channels=ch,
                        d_state=n, groups=1, softplus=1, type=L.BF16)
        check(lib().b200_op_ssm_scan(C.byref(c), None, 0, None))
        return [v.clone() for v in (d["y"], s, t)]

    near = run(0, 0)
    for far in (run((1 << 31) // (rows - 1) + 8, 0), run(0, (1 << 31) // 2 + 8)):
        for p, q in zip(near, far):
            assert torch.equal(p, q)


def test_selection():
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(6, 1000, generator=g, device="cuda").to(torch.float16)
    score, slot = torch.rand(6, generator=g, device="cuda"), torch.arange(6, dtype=torch.int32, device="cuda")
    found = []
    for rows in (logits, spread(logits, (1 << 31) // 4 + 1)):
        to = [torch.zeros(10, dtype=torch.float32 if i == 0 else torch.int32, device="cuda") for i in range(4)]
        a = BeamSelectArgs(logits=rows.data_ptr(), logits_stride=rows.stride(0), score=score.data_ptr(), slot=slot.data_ptr(), to_score=to[0].data_ptr(), to_beam=to[1].data_ptr(),
                           to_token=to[2].data_ptr(), to_slot=to[3].data_ptr(), n_requests=2, n_beams=3, n_vocab=1000, n_keep=5, type=L.F16)
        ws = torch.empty(lib().b200_beam_select_workspace_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
        check(lib().b200_op_beam_select(C.byref(a), ws.data_ptr(), ws.numel(), None))
        found.append(to)
    assert torch.equal(found[0][1], found[1][1]) and torch.equal(found[0][2], found[1][2]) and torch.equal(found[0][3], found[1][3])
    assert np.allclose(found[0][0].cpu(), found[1][0].cpu(), rtol=1e-6)  # (lanes add up other tokens where rows begin on 16 bytes)


def test_reordering():
    x = torch.arange(4 * 100, dtype=torch.int32, device="cuda").reshape(4, 100)
    far = spread(x, (1 << 31) // 4 + 12)
    src, dst = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([1, 2, 3, 0], [0, 1, 2, 3]))
    s = (SlotState * 1)(SlotState(far.data_ptr(), 4 * far.stride(0), 400))
    check(lib().b200_op_state_reorder(s, 1, src.data_ptr(), dst.data_ptr(), 4, 4, None, None))
    assert torch.equal(far, x[[1, 2, 3, 0]])
