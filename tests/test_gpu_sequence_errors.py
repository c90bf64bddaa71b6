"""Batch steps that are refused leave every sequence as it was, over f32 caches by cell and over pages in 8 bits (include/b200_llama.h, b200_llama_decode_batch)."""
import ctypes as C

import numpy as np
import pytest
import torch

import galirax_ref as R
from koboldcpp_b200 import galirax as G
from koboldcpp_b200.lib import B200Error, Kv8Map, check, lib

pytestmark = pytest.mark.gpu

CONFIG = R.make_config([R.lightning_layer(heads=2, dim=16, vdim=32, mlp=None), R.attn_layer(heads=4, kv_heads=2, dim=32, vdim=48, rot_dims=16, mlp=None)], width=64, vocab=70)


def without_a_buffer(model, tokens, seqs):
    """A step that wants logits and has nowhere to put them."""
    t, s, w = np.array(tokens, np.int32), np.array(seqs, np.int32), np.ones(len(tokens), np.int8)
    assert lib().b200_llama_decode_batch(model.h, t.ctypes.data, s.ctypes.data, w.ctypes.data, len(t), None) == 2


@pytest.mark.parametrize("kv8_page", [0, 16])
def test_a_step_without_room_for_its_logits(kv8_page):
    W = R.as_tensors(R.random_weights(CONFIG, seed=5))
    toks = np.random.default_rng(3).integers(0, CONFIG["vocab"], 60).tolist()
    runs = []
    for refused in (False, True):
        m = G.build(CONFIG, W, dtype="float32", n_ctx=256, n_seq_max=3, max_batch=64, kv8_page=kv8_page)
        a, b = m.seq_open(), m.seq_open()
        if refused:
            without_a_buffer(m, toks[:20], [a] * 20)  # its first tokens: the recurrent layers' state begins with the next step
        assert m.seq_length(a) == 0
        rows = [m.decode_batch(toks[:20], [a] * 20, [1] * 20)]
        if refused:
            without_a_buffer(m, toks[20:40] + [1, 2], [a] * 20 + [b] * 2)
        assert (m.seq_length(a), m.seq_length(b)) == (20, 0)
        rows.append(m.decode_batch(toks[20:41] + toks[:9], [a] * 21 + [b] * 9, [1] * 30))
        if refused:
            without_a_buffer(m, [1], [b])
        rows.append(m.decode_batch(toks[41:42] + toks[9:10], [a, b], [1, 1]))
        assert (m.seq_length(a), m.seq_length(b)) == (42, 10)
        with pytest.raises(B200Error, match="full"):
            for _ in range(4):
                m.decode_batch([1] * 64, [a] * 64, [0] * 64)
        m.seq_close(a)
        rows.append(m.decode_batch(toks[10:20], [b] * 10, [1] * 10))
        runs.append(np.concatenate(rows))
        m.close()
    assert np.array_equal(runs[0], runs[1])


def test_refused_rows_are_counted_in_pinned_host_memory():
    """The place where the decoder has them counted."""
    table, length, refs = torch.full((2, 4), -1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    count = torch.zeros(64, dtype=torch.int32).pin_memory()
    rows, new = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    ws = torch.zeros(lib().b200_kv8_grow_workspace_bytes(2), dtype=torch.uint8, device="cuda")
    m = Kv8Map(table.data_ptr(), 4, length.data_ptr(), refs.data_ptr(), 2, 3, 16)
    for want in (1, 2):
        check(lib().b200_op_kv8_grow(C.byref(m), None, 0, rows.data_ptr(), new.data_ptr(), 2, None, count[5:].data_ptr(), ws.data_ptr(), ws.numel(), None))
        torch.cuda.synchronize()
        assert count.tolist() == [0] * 5 + [1 if want == 1 else 3] + [0] * 58
    assert length.tolist() == [40, 0]
