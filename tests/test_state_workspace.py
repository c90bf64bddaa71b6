"""How much workspace scans ask for (include/b200_state.h), without a GPU: what a step of any make-up needs is bounded, and follows what is cut in stretches, not how many sequences there are."""
import ctypes as C
import random
import re

import pytest

from koboldcpp_b200.lib import lib
from test_state_host import AT, HEADER, INVALID, scan_args


def room(n_seq, n_tokens, max_new, channels, d_state=16, groups=1):
    a = scan_args(n_seq=n_seq, n_slots=n_seq, n_tokens=n_tokens, max_new=max_new, channels=channels, d_state=d_state, groups=groups, slot_stride=channels * d_state)
    return lib().b200_ssm_scan_workspace_bytes(C.byref(a))


def most():
    m = re.search(r"#define B200_SSM_SCAN_WORKSPACE_MAX \(1 << (\d+)\)", HEADER.read_text())
    return 1 << int(m.group(1))


@pytest.mark.parametrize("singles,prompt", [(96, 4096), (128, 2048), (64, 2048), (1, 4096), (300, 4096)])
@pytest.mark.parametrize("max_new", [True, False])
def test_single_rows_beside_a_prompt(singles, prompt, max_new):
    """8192 channels of 16 states, 512 KB a state: the single rows take no places."""
    size = room(singles + 1, singles + prompt, prompt if max_new else 0, 8192)
    assert size <= 1.25 * room(2, singles + prompt, 0, 8192)  # (several sequences are cut in more stretches than one)
    assert size <= most()


def test_no_step_needs_more_than_the_header_says():
    rng = random.Random(0)
    largest = 0
    for _ in range(200000):
        channels, d_state = rng.choice([1, 37, 64, 128, 129, 1024, 2048, 2560, 5120, 8192, 12000, 16384, 23000, int(2 ** rng.uniform(0, 18))]), rng.choice([1, 2, 8, 15, 16, 17, 32, 33, 64, 65, 128, rng.randint(1, 128)])
        tokens = int(2 ** rng.uniform(0, 22))
        size = room(rng.choice([1, 2, 3, 7, 64, 1000, 65535]), tokens, rng.choice([0, rng.randint(1, tokens), max(1, tokens // rng.randint(1, 9))]), channels, d_state,
                    rng.choice([g for g in (1, 2, 4, 8, channels) if channels % g == 0]))
        largest = max(largest, size)
        assert size <= most()
    assert largest > most() // 4  # (a bound that says something)


def test_a_workspace_of_that_size_is_enough_for_every_step():
    """Sized once: a step that asks for more than another, larger one is not refused.  (Kept from the device by a result that is not aligned, which is looked at before; then by a workspace one byte short.)"""
    for tokens in (500, 4096, 100000):
        a = scan_args(n_tokens=tokens, channels=2048, slot_stride=1 << 20, x_stride=2048, dt_stride=2048, z_stride=2048, dst_stride=2048)
        need = lib().b200_ssm_scan_workspace_bytes(C.byref(a))
        assert 0 < need <= most()
        assert lib().b200_op_ssm_scan(C.byref(a), AT, need - 1, None) == INVALID
        assert str(need).encode() in lib().b200_last_error()
