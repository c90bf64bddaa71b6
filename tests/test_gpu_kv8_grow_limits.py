"""b200_op_kv8_grow where sums over the rows of a call pass 31 bits (include/b200_kv8.h)."""
import ctypes as C

import pytest
import torch

from koboldcpp_b200.lib import Kv8Map, check, lib

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


def grow(table, length, refs, rows, new, page=16, with_info=True):
    n = len(rows)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    r, m, refused, info = ints(rows), ints(new), ints([0]), torch.full((4, n), -9, dtype=torch.int32, device="cuda")
    ws = torch.zeros(lib().b200_kv8_grow_workspace_bytes(n), dtype=torch.uint8, device="cuda")
    c_map = Kv8Map(table.data_ptr(), table.shape[1], length.data_ptr(), refs.data_ptr(), table.shape[0], refs.numel(), page)
    check(lib().b200_op_kv8_grow(C.byref(c_map), None, 0, r.data_ptr(), m.data_ptr(), n, info.data_ptr() if with_info else None, refused.data_ptr(), ws.data_ptr(), ws.numel(), None))
    return info.tolist(), int(refused)


def small_map(n_rows=5, n_pages=20):
    return (torch.full((n_rows, 6), -1, dtype=torch.int32, device="cuda"), torch.zeros(n_rows, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda"))


def test_rows_behind_more_tokens_than_a_step_can_have():
    table, length, refs = small_map()
    info, refused = grow(table, length, refs, [0, 1, 2, 3, 4], [5, MOST, 7, MOST, 9])  # rows 1 and 3 do not fit their table; rows 2 and 4 would begin behind 2^31 - 1
    assert info == [[0, 5, MOST, MOST, MOST], [5, 0, 0, 0, 0], [0, 1, 2, 3, 4], [0, 0, 0, 0, 0]]
    assert refused == 4 and length.tolist() == [5, 0, 0, 0, 0] and refs.tolist() == [1] + [0] * 19
    assert table.tolist() == [[0, -1, -1, -1, -1, -1]] + [[-1] * 6] * 4


def test_the_last_place_there_is():
    table, length, refs = small_map()
    info, refused = grow(table, length, refs, [0, 1, 2], [MOST - 9, 9, 1])
    assert info == [[0, MOST - 9, MOST], [0, 9, 0], [0, 1, 2], [0, 0, 0]] and refused == 2 and length.tolist() == [0, 9, 0, 0, 0]


def test_without_a_step_there_are_no_places():
    table, length, refs = small_map()
    _, refused = grow(table, length, refs, [0, 1, 2], [5, MOST, 7], with_info=False)
    assert refused == 1 and length.tolist() == [5, 0, 7, 0, 0]


def test_more_pages_asked_for_than_31_bits_hold():
    """33 rows of 2^26 pages each, one that asks for little in front of them and one behind: a table of 9 GB."""
    n, pages = 33, 2 ** 26
    table = torch.full((n + 2, pages), -1, dtype=torch.int32, device="cuda")
    length, refs = torch.zeros(n + 2, dtype=torch.int32, device="cuda"), torch.zeros(50, dtype=torch.int32, device="cuda")
    _, refused = grow(table, length, refs, [n, *range(n), n + 1], [20, *[pages * 16] * n, 20], with_info=False)
    assert refused == n + 1  # (what is asked for by a refused row counts against those behind it)
    assert length.tolist() == [0] * n + [20, 0] and refs.tolist() == [1, 1] + [0] * 48
    assert table[:, :4].tolist() == [[-1] * 4] * n + [[0, 1, -1, -1], [-1] * 4]
    assert int((table >= 0).sum()) == 2
