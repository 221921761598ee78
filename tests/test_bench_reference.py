"""bench.py --impl reference: the reference cannot run on the machines that the benchmark runs on, and nothing of this library stands in
for it."""
import json
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_reference_arm_says_that_it_is_not_to_be_had():
    r = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--gpus", "1", "--steps", "2", "--warmup", "1"], cwd=ROOT, stdout=subprocess.PIPE, text=True, timeout=300)
    assert r.returncode == 0
    line = json.loads(r.stdout)
    assert set(line) == {"impl", "unavailable"} and line["impl"] == "reference"
    assert "\n" not in line["unavailable"] and len(line["unavailable"]) > 20


def test_other_ranks_are_silent():
    env = dict(os.environ, RANK="1", WORLD_SIZE="2", LOCAL_RANK="1")
    r = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--gpus", "2", "--steps", "2", "--warmup", "1"], cwd=ROOT, env=env, stdout=subprocess.PIPE, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == ""
