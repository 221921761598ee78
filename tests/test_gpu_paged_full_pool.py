"""The serving loop of examples/paged_step.py where the pool has too few pages for its chats: what it takes a chat to hold is what the
plans served, and no chat's rows come to lie on another's page."""
import importlib.util
import os

import pytest
import torch

import q4gpu
from gpu_util import lib

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "paged_step.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_step", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
def test_loop_goes_on_where_pages_run_out(example, kind):
    L = lib()
    L.q4_gpu_last_error()
    loop = example.Loop(1, 9, n_pages=40, kind=q4gpu.KIND_Q8 if kind == "q8_0" else q4gpu.KIND_F16, seed=3)
    pool = loop.pool
    plan, append, trim = pool.plan, pool.append, pool.trim
    rows_of = [torch.empty(0, 256, device="cuda") for _ in range(9)]   # K of the rows that each place holds
    short = [0]

    def planned(rows, add, *maps):
        assert rows.tolist() == [len(x) for x in rows_of]              # what the loop says is what was served so far
        plan(rows, add, *maps)
        short[0] += int(loop.start[-1]) < int(add.sum())

    def appended(layer, k, v, slot):
        append(layer, k, v, slot)
        start = loop.start.tolist()
        for r in range(9):
            rows_of[r] = torch.cat([rows_of[r], k[start[r]: start[r + 1]]])
        table = loop.table
        for r, x in enumerate(rows_of):                                # every row of every place is still there
            if len(x):
                p = torch.arange(len(x), device="cuda")
                got = torch.empty_like(x)
                pool.gather(0, (table[r].long()[p // 64] * 64 + p % 64).int(), got, None)
                # codes are half of amax / 127 off, their scale 2^-11 of itself (127 codes of it: 0.06); fp16: 2^-11
                assert ((got - x).abs() <= 0.6 / 127 * x.abs().max()).all()

    def trimmed(rows, keep, table):
        assert rows.tolist() == [len(x) for x in rows_of]
        trim(rows, keep, table)
        for r, n in enumerate(keep.tolist()):
            rows_of[r] = rows_of[r][:n]

    pool.plan, pool.append, pool.trim = planned, appended, trimmed
    tokens = sum(loop.step(check=i % 10 == 0) for i in range(60))
    assert short[0] > 0 and tokens > 2000
    pool.plan, pool.append, pool.trim = plan, append, trim
    assert loop.end() and L.q4_gpu_last_error() == 0


def test_command_with_few_pages(example, capsys):
    assert example.main(["--layers", "2", "--chats", "9", "--steps", "40", "--check", "4", "--pages", "36"]) == 0
    assert "10 steps checked; status 0; pages back: True" in capsys.readouterr().out
