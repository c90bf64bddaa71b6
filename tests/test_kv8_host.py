"""The paged 8-bit cache without a GPU: what the calls refuse, sizes, and the reference that the GPU tests compare with."""
import ctypes as C
import re
from pathlib import Path

import numpy as np
import pytest

import kv8_ref as R
import koboldcpp_b200.lib as L
from koboldcpp_b200.lib import Kv8AttnArgs, Kv8Cache, Kv8LoadArgs, Kv8Map, Kv8StoreArgs, lib

HEADER = Path(__file__).resolve().parent.parent / "include" / "b200_kv8.h"
AT = 4096  # an address that is never read: every call below ends before it would be


def test_every_symbol_is_exported_and_bound():
    declared = set(re.findall(r"B200_API\s+[\w\s\*]+?\b(b200_\w+)\s*\(", HEADER.read_text()))
    assert declared == set(L._KV8_SIGS)
    for name in declared:
        assert hasattr(lib(), name)


def test_structures_have_the_header_s_layout(tmp_path):
    """Offsets of every field as the C compiler has them."""
    import subprocess
    names = {"b200_kv8_cache": Kv8Cache, "b200_kv8_store_args": Kv8StoreArgs, "b200_kv8_load_args": Kv8LoadArgs, "b200_kv8_attn_args": Kv8AttnArgs, "b200_kv8_map": Kv8Map}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "p.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "p")], check=True)
    for line in subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, value = line.split()
        c, _, f = name.partition(".")
        assert int(value) == (getattr(names[c], f).offset if f else C.sizeof(names[c])), name


@pytest.mark.parametrize("page,heads,dim,vdim", [(16, 8, 128, 128), (32, 1, 64, 64), (64, 3, 96, 80), (128, 32, 256, 16)])
def test_page_bytes(page, heads, dim, vdim):
    assert lib().b200_kv8_page_bytes(page, heads, dim, vdim) == R.Pool(1, page, heads, dim, vdim).bytes


@pytest.mark.parametrize("page,heads,dim,vdim", [(8, 8, 128, 128), (48, 8, 128, 128), (256, 8, 128, 128), (16, 0, 128, 128), (16, 1025, 128, 128), (16, 8, 120, 128), (16, 8, 0, 128), (16, 8, 272, 128),
                                                 (16, 8, 128, 8), (16, 8, 128, 272), (-16, 8, 128, 128)])
def test_sizes_that_no_cache_has(page, heads, dim, vdim):
    assert lib().b200_kv8_page_bytes(page, heads, dim, vdim) == 0
    a = Kv8StoreArgs(Kv8Cache(AT, 4, page, heads, dim, vdim), AT, 1 << 20, AT, 1 << 20, AT, AT, 4, 1, 1, 1, L.F32)
    assert lib().b200_op_kv8_store(C.byref(a), None) == 1


def store_args(kind, **change):
    f = dict(cache=Kv8Cache(AT, 4, 16, 2, 64, 64), k=AT, k_stride=128, v=AT, v_stride=128, seq_info=AT, table=AT, table_stride=4, n_rows=1, n_seq=1, n_tokens=1, type=L.F32)
    f.update(change)
    return kind(*[f[name] for name, _ in kind._fields_])


COMMON = [(dict(cache=Kv8Cache(None, 4, 16, 2, 64, 64)), 2), (dict(cache=Kv8Cache(AT + 8, 4, 16, 2, 64, 64)), 2), (dict(cache=Kv8Cache(AT, 0, 16, 2, 64, 64)), 2), (dict(seq_info=None), 2),
          (dict(table=None), 2), (dict(n_seq=-1), 2), (dict(n_tokens=-1), 2), (dict(n_rows=-1), 2), (dict(table_stride=-1), 2), (dict(table_stride=1 << 30), 1), (dict(n_seq=1025), 1),
          (dict(type=L.Q8_0), 1), (dict(seq_info=AT + 2), 2), (dict(table=AT + 1), 2)]


@pytest.mark.parametrize("change,code", COMMON + [(dict(k=None), 2), (dict(v=None), 2), (dict(k_stride=127), 2), (dict(v_stride=0), 2), (dict(k=AT + 2), 2), (dict(v=AT + 1), 2)])
def test_store_refuses(change, code):
    assert lib().b200_op_kv8_store(C.byref(store_args(Kv8StoreArgs, **change)), None) == code
    assert b"b200_op_kv8_store" in lib().b200_last_error()


@pytest.mark.parametrize("change,code", COMMON + [(dict(k_stride=127), 2), (dict(v_stride=0), 2), (dict(k=AT + 1), 2)])
def test_load_refuses(change, code):
    assert lib().b200_op_kv8_load(C.byref(store_args(Kv8LoadArgs, **change)), None) == code
    assert b"b200_op_kv8_load" in lib().b200_last_error()


def attn_args(**change):
    f = dict(cache=Kv8Cache(AT, 4, 16, 2, 64, 64), q=AT, q_stride=256, dst=AT, dst_stride=256, seq_info=AT, table=AT, table_stride=4, n_rows=1, n_seq=1, n_tokens=1, max_new=1, n_head=4, type=L.F32,
             sink=None, window=0, keep_first=0, scale=1.0, softcap=0.0, f16_products=0)
    f.update(change)
    return Kv8AttnArgs(*[f[name] for name, _ in Kv8AttnArgs._fields_])


@pytest.mark.parametrize("change,code", COMMON + [(dict(q=None), 2), (dict(dst=None), 2), (dict(q_stride=255), 2), (dict(dst_stride=1), 2), (dict(n_head=0), 2), (dict(n_head=5), 2), (dict(n_tokens=1 << 28, n_head=8, q_stride=512, dst_stride=512), 1),
                                                  (dict(q=AT + 2), 2), (dict(dst=AT + 1), 2), (dict(sink=AT + 2), 2), (dict(window=-1), 2),
                                                  (dict(keep_first=-1), 2), (dict(softcap=-1.0), 2), (dict(softcap=float("nan")), 2), (dict(softcap=float("inf")), 2), (dict(scale=float("nan")), 2)])
def test_attn_refuses(change, code):
    assert lib().b200_op_kv8_attn(C.byref(attn_args(**change)), AT, 1 << 30, None) == code
    assert b"b200_op_kv8_attn" in lib().b200_last_error()


def test_attn_refuses_a_workspace_that_is_none():
    a = attn_args()
    need = lib().b200_kv8_attn_workspace_bytes(C.byref(a))
    assert need > 0
    for ws, size in ((None, need), (AT, need - 1), (AT + 8, need)):
        assert lib().b200_op_kv8_attn(C.byref(a), ws, size, None) == 2


def test_attn_refuses_a_limit_below_zero():
    assert lib().b200_op_kv8_attn_wait(C.byref(attn_args()), AT, 1 << 30, -1, None) == 2


def test_calls_without_work_touch_nothing():
    for change in (dict(n_tokens=0), dict(n_seq=0)):
        assert lib().b200_op_kv8_store(C.byref(store_args(Kv8StoreArgs, k=None, v=None, seq_info=None, table=None, **change)), None) == 0
        assert lib().b200_op_kv8_load(C.byref(store_args(Kv8LoadArgs, seq_info=None, table=None, **change)), None) == 0
        assert lib().b200_op_kv8_attn(C.byref(attn_args(q=None, dst=None, seq_info=None, table=None, **change)), None, 0, None) == 0
    m = Kv8Map(AT, 4, AT, AT, 2, 4, 16)
    assert lib().b200_op_kv8_cut(C.byref(m), None, None, 0, None) == 0
    assert lib().b200_op_kv8_fork(C.byref(m), None, None, 0, None, None) == 0
    assert lib().b200_op_kv8_grow(C.byref(m), None, 0, None, None, 0, None, None, None, 0, None) == 0
    assert lib().b200_op_kv8_copy_pages(None, 0, None, None, 3, None) == 0


def test_page_calls_refuse():
    ll, good, cache = lib(), dict(table=AT, table_stride=4, len=AT, refs=AT, n_rows=2, n_pages=4, page_size=16, _pad=0), (Kv8Cache * 1)(Kv8Cache(AT, 4, 16, 2, 64, 64))

    def mapping(**change):
        return C.byref(Kv8Map(*[{**good, **change}[name] for name, _ in Kv8Map._fields_]))

    for change, code in ((dict(table=None), 2), (dict(len=None), 2), (dict(refs=None), 2), (dict(n_rows=0), 2), (dict(n_pages=0), 2), (dict(table_stride=0), 2), (dict(page_size=20), 1),
                         (dict(table_stride=1 << 29), 1)):
        m = mapping(**change)
        assert ll.b200_op_kv8_cut(m, AT, None, 1, None) == code, change
        assert ll.b200_op_kv8_fork(m, AT, AT, 1, None, None) == code, change
        assert ll.b200_op_kv8_grow(m, cache, 1, AT, AT, 1, None, None, AT, 1 << 20, None) == code, change
        assert ll.b200_op_kv8_compact(m, cache, 1, None, AT, 1 << 20, None) == code, change
    m = mapping()
    for n, code in ((-1, 2), (1025, 1)):
        assert ll.b200_op_kv8_cut(m, AT, None, n, None) == code
        assert ll.b200_op_kv8_fork(m, AT, AT, n, None, None) == code
        assert ll.b200_op_kv8_grow(m, cache, 1, AT, AT, n, None, None, AT, 1 << 20, None) == code
    assert ll.b200_op_kv8_cut(m, None, None, 1, None) == 2
    assert ll.b200_op_kv8_fork(m, None, AT, 1, None, None) == 2 and ll.b200_op_kv8_fork(m, AT, None, 1, None, None) == 2
    assert ll.b200_op_kv8_grow(m, cache, 1, None, AT, 1, None, None, AT, 1 << 20, None) == 2 and ll.b200_op_kv8_grow(m, cache, 1, AT, None, 1, None, None, AT, 1 << 20, None) == 2
    assert ll.b200_op_kv8_grow(m, cache, 1, AT, AT, 1, None, None, None, 0, None) == 2 and ll.b200_op_kv8_grow(m, cache, 1, AT, AT, 1, None, None, AT, 7, None) == 2
    assert ll.b200_op_kv8_grow(m, cache, 1, AT, AT, 1, None, None, AT + 4, 1 << 20, None) == 2
    need = ll.b200_kv8_compact_workspace_bytes(4)
    assert need > 0 and ll.b200_op_kv8_compact(m, cache, 1, None, AT, need - 1, None) == 2 and ll.b200_op_kv8_compact(m, cache, 1, None, None, need, None) == 2
    for bad, code in ((Kv8Cache(AT, 3, 16, 2, 64, 64), 2), (Kv8Cache(AT, 4, 32, 2, 64, 64), 2), (Kv8Cache(None, 4, 16, 2, 64, 64), 2), (Kv8Cache(AT, 4, 16, 2, 60, 64), 1)):
        one = (Kv8Cache * 1)(bad)
        assert ll.b200_op_kv8_grow(m, one, 1, AT, AT, 1, None, None, AT, 1 << 20, None) == code
        assert ll.b200_op_kv8_compact(m, one, 1, None, AT, 1 << 20, None) == code
    assert ll.b200_op_kv8_grow(m, None, 1, AT, AT, 1, None, None, AT, 1 << 20, None) == 2
    assert ll.b200_op_kv8_copy_pages(cache, 1, None, AT, 1, None) == 2 and ll.b200_op_kv8_copy_pages(cache, 1, AT, AT, -1, None) == 2 and ll.b200_op_kv8_copy_pages(None, 2, AT, AT, 1, None) == 2


def test_no_gpu_means_an_error():
    if lib().b200_device_count() > 0:
        pytest.skip("a GPU is present")
    assert lib().b200_op_kv8_store(C.byref(store_args(Kv8StoreArgs)), None) == 3
    assert lib().b200_op_kv8_cut(C.byref(Kv8Map(AT, 4, AT, AT, 2, 4, 16)), AT, None, 1, None) == 3


# ------------------------------------------------------------------------------------------------ the reference itself
def test_reference_stays_within_the_stated_error():
    """A page filled in one call is off by half a step of its scale at most (the scale is a / 127 rounded to f32, so a value may lie 2^-24 of itself, 127 2^-24 steps,
    beyond 127 and is clamped); one that fills token by token by 2.5 steps of its last scale: half a step for the value, half a step of the scale of the
    time for every growth, and those scales are 0.8, 0.64, ... of the last one: 0.5 (1 + 0.8 + 0.64 + ..) = 2.5."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((16, 2, 64)) * np.exp(0.5 * rng.standard_normal((16, 1, 1)))
    pool = R.Pool(2, 16, 2, 64, 64)
    pool.store([1], x, x, 0)
    got, _ = pool.rows([1], 16, "k")
    assert (np.abs(got - x) <= pool.ks[1][:, None] * (0.5 + 127 * 2.0 ** -24)).all()
    louder = x * np.linspace(0.2, 3, 16)[:, None, None]
    for t in range(16):
        pool.store([0], louder[t:t + 1], louder[t:t + 1], t)
    got, _ = pool.rows([0], 16, "v")
    assert (np.abs(got - louder) <= pool.vs[0][:, None] * (2.5 + 127 * 2.0 ** -24)).all()


def test_reference_softmax_by_hand():
    pool = R.Pool(1, 16, 1, 16, 16)
    pool.put(np.zeros((1, 1, 16, 16)), np.arange(16)[None, None, :, None] * np.ones((1, 1, 16, 16)), np.ones((1, 1)), np.full((1, 1), 0.5))
    out, _, _ = pool.attend([0], np.ones((1, 1, 16)), 3, 1.0)
    assert np.allclose(out, 0.5 * (0 + 1 + 2 + 3) / 4)  # equal scores over four keys
    out, _, _ = pool.attend([0], np.ones((1, 1, 16)), 3, 1.0, sink=np.zeros(1))
    assert np.allclose(out, 0.5 * (0 + 1 + 2 + 3) / 5)
    out, _, _ = pool.attend([0], np.ones((1, 1, 16)), 9, 1.0, window=2, keep=1)
    assert np.allclose(out, 0.5 * (0 + 8 + 9) / 3)
    out, _, _ = pool.attend([-1], np.ones((1, 1, 16)), 3, 1.0)
    assert (out == 0).all()


def test_reference_pages():
    m = R.Pages(4, 4, 8, 16)
    info, refused, copies = m.grow([2, 0], [20, 5])
    assert refused == 0 and copies == [] and m.table[2, :2].tolist() == [0, 1] and m.table[0, 0] == 2 and info.tolist() == [[0, 20], [20, 5], [2, 0], [0, 0]]
    assert m.fork([2, 2, 9], [1, 3, 0]) == 1 and m.refs[:3].tolist() == [3, 3, 1]
    _, refused, copies = m.grow([1, 3], [1, 1])
    assert refused == 0 and copies == [(1, 3), (1, 4)] and m.refs.tolist() == [3, 1, 1, 1, 1, 0, 0, 0]
    m.cut([2], None)
    assert m.refs.tolist() == [2, 0, 1, 1, 1, 0, 0, 0]
    assert m.compact() == (4, [(4, 1)]) and m.table[3, :2].tolist() == [0, 1] and m.table[1, :2].tolist() == [0, 3]
    assert m.grow([0, 0, 1], [70, 1, 400])[1] == 3  # beyond the table; named twice; beyond the table


def test_other_architectures_refuse_pages(tmp_path):
    import json
    from koboldcpp_b200 import models
    (tmp_path / "config.json").write_text(json.dumps({"architecture": "Zevopel"}))
    with pytest.raises(L.B200Error, match="8-bit pages"):
        models.load_model(tmp_path, kv8_page=16)
