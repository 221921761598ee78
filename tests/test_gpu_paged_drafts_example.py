"""The serving loop with drafts of examples/paged_drafts.py: plan, prep, attend, verify, release, forks of shared instructions and compaction together, with its own checks on."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_drafts.py")


@pytest.mark.parametrize("args", [["--kind", "q8_0"], ["--kind", "f16", "--drafts", "7", "--chats", "3"], ["--temp", "0", "--drafts", "2"], ["--drafts", "0", "--chats", "5"], ["--steps", "90", "--drafts", "6", "--chats", "4", "--check", "30"]])
def test_a_serving_loop_with_drafts(args, capsys):
    spec = importlib.util.spec_from_file_location("paged_drafts", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(["--layers", "2", "--steps", "15", "--check", "5"] + args) == 0
    assert "3 steps checked; status 0; pages back: True" in capsys.readouterr().out
