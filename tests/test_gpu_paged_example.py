"""The serving loop of examples/paged_step.py: chats that come and go, checked in 64 bits as it runs."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "paged_step.py")


@pytest.mark.parametrize("kind", ["q8_0", "f16"])
def test_paged_serving_loop(kind, capsys):
    spec = importlib.util.spec_from_file_location("paged_step", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(["--layers", "2", "--chats", "9", "--steps", "30", "--check", "3", "--kind", kind]) == 0
    assert "10 steps checked; status 0; pages back: True" in capsys.readouterr().out
