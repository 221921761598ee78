"""The paged KV cache (q4_gpu_pages_*) at its limits: tables whose entries are no pages, statuses, places without tokens, scratch that is
not to be had."""
import pytest
import torch

import q4gpu
from gpu_util import lib
from test_gpu_pages import KINDS, Step, attend_exact, ints, plan_plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [-1, -2**31, "n_pages", 2**31 - 1])
@pytest.mark.parametrize("rows,keep,at", [([70, 33], [0, 0], (1, 2)), ([70, 33], [17, 40], (0, 4)), ([16 * 300] + [5] * 2000, [0] * 2001, (0, 299)),
                                          ([16 * 300] + [5] * 2000, [0] * 2001, (2000, 0))])
def test_trim_refuses_entries_that_are_no_pages(rows, keep, at, bad):
    """nothing goes back, whatever the other entries are; a plan behind it gets pages of the pool only"""
    s = Step(rows, [0] * len(rows))
    bad = s.pool.n_pages if bad == "n_pages" else bad
    free = s.free_now()
    L = lib()
    L.q4_gpu_last_error()
    table = s.d_table.clone()
    table[at] = bad
    s.pool.trim(s.d_rows, ints(keep), table)
    assert L.q4_gpu_last_error() == 4
    assert s.free_now() == free
    s.pool.trim(s.d_rows, ints(keep), s.d_table)          # the right table: all of them, and each once
    assert L.q4_gpu_last_error() == 0
    held = sum(-(-max(k, 0) // 16) if k < h else -(-h // 16) for h, k in zip(rows, keep))
    now = s.free_now()
    assert len(now) == s.pool.n_pages - held and len(set(now)) == len(now) and min(now) >= 0 and max(now) < s.pool.n_pages


def test_trim_does_not_look_at_entries_that_stay():
    s = Step([70, 33], [0, 0])
    table = s.d_table.clone()
    table[0, 0], table[1, 2] = -1, -1                     # page 0 of the first is kept, as all of the second's are
    lib().q4_gpu_last_error()
    s.pool.trim(s.d_rows, ints([5, 33]), table)
    assert lib().q4_gpu_last_error() == 0
    assert s.free_now() == s.free + s.table[0][1:5][::-1]
