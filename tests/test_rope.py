"""Frequencies of a rotation (q4_gpu_rope_set, on the host): against the formulas, whatever the position; what is refused."""
import math
from fractions import Fraction

import pytest

import q4gpu

TWO_PI = Fraction(6283185307179586476925286766559005768394, 10**39)


def wanted(n_rot, base, scaling=None, factor=1.0, orig=0.0, fast=32.0, slow=1.0):
    """radians per position, from the definition"""
    n = n_rot // 2
    out = []
    for i in range(n):
        f = base ** (-2 * i / n_rot)
        s = 0.0
        if scaling == "linear":
            s = 1.0
        elif scaling == "ramp":
            lo = max(0, math.floor(n * math.log(orig / (fast * 2 * math.pi)) / math.log(base)))
            hi = min(n - 1, math.ceil(n * math.log(orig / (slow * 2 * math.pi)) / math.log(base)))
            s = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
        elif scaling == "smooth":
            s = 1 - min(1.0, max(0.0, (f * orig / (2 * math.pi) - slow) / (fast - slow)))
        out.append(f * (1 - s) + f / factor * s)
    return out


@pytest.mark.parametrize("n_rot,base", [(2, 10000.0), (64, 1e7), (128, 1e6), (256, 5e5), (6, 10.0), (0, 1e4)])
@pytest.mark.parametrize("scaling", [None, dict(scaling="linear", factor=4.0), dict(scaling="ramp", factor=8.0, orig=8192), dict(scaling="ramp", factor=40.0, orig=4096, fast=16.0, slow=2.0),
                                     dict(scaling="smooth", factor=8.0, orig=8192, fast=4.0, slow=1.0), dict(scaling="linear", factor=0.01)])
def test_turns(n_rot, base, scaling):
    r = q4gpu.Rope(n_rot, base, **(scaling or {}))
    assert (r.n_rot, r.half, r.mag) == (n_rot, 0, 1.0)
    for i, f in enumerate(wanted(n_rot, base, **(scaling or {}))):
        # a frequency is computed in 64 bits: pow, the ramp and the division by 2 pi are off by 2^-50 of it at most, and what is kept of a turn by 2^-53
        off = (Fraction(r.turn[i], 2**64) - Fraction(f) / TWO_PI) % 1
        off = min(off, 1 - off)
        assert off <= Fraction(f) / 2**49 + Fraction(1, 2**52)
    assert all(t == 0 for t in r.turn[n_rot // 2:])


def test_angles_of_far_positions():
    r = q4gpu.Rope(64, 1e7)
    for i, f in enumerate(wanted(64, 1e7)):
        for pos in (1, 77, 262143, 2**31 - 1):
            angle = Fraction((pos * r.turn[i]) % 2**64, 2**64)
            off = (angle - Fraction(f) * pos / TWO_PI) % 1
            assert min(off, 1 - off) <= pos * (Fraction(f) / 2**49 + Fraction(1, 2**52))


def test_the_whole_descriptor():
    r = q4gpu.Rope(32, 1e4, half=True, mag=1.25)
    assert (r.n_rot, r.half, r.mag, r.reserved) == (32, 1, 1.25, 0)


@pytest.mark.parametrize("args", [
    dict(n_rot=3, base=1e4), dict(n_rot=258, base=1e4), dict(n_rot=-2, base=1e4), dict(n_rot=12, base=1e4, half=True), dict(n_rot=8, base=0.0), dict(n_rot=8, base=-5.0),
    dict(n_rot=8, base=float("nan")), dict(n_rot=8, base=float("inf")), dict(n_rot=8, base=1e4, mag=0.0), dict(n_rot=8, base=1e4, mag=float("nan")), dict(n_rot=8, base=1e4, mag=1e39),
    dict(n_rot=8, base=1e4, scaling="linear", factor=0.0), dict(n_rot=8, base=1e4, scaling="linear", factor=float("nan")), dict(n_rot=8, base=1e4, scaling="other"),
    dict(n_rot=8, base=1e4, scaling="ramp", factor=2.0), dict(n_rot=8, base=1.0, scaling="ramp", factor=2.0, orig=100), dict(n_rot=8, base=1e4, scaling="ramp", factor=2.0, orig=100, fast=1.0, slow=1.0),
    dict(n_rot=8, base=1e4, scaling="smooth", factor=2.0, orig=100, fast=4.0, slow=0.0), dict(n_rot=256, base=1e-300, scaling="linear", factor=1e-300)])
def test_refusals(args):
    with pytest.raises(RuntimeError):
        q4gpu.Rope(**args)
    q4gpu.load().q4_gpu_last_error()


def ramp(n_rot, base, factor, orig, fast, slow):
    """radians per position by the definition of the ramp: it ends at the pair that turns `slow` times, which may lie behind the last one; no later than at n_rot - 1"""
    def pair(turns):                                       # base^(-2 i / n_rot) * orig = 2 pi turns
        return n_rot * (math.log(orig) - math.log(2 * math.pi * turns)) / (2 * math.log(base))
    lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), n_rot - 1)
    f = [base ** (-2 * i / n_rot) for i in range(n_rot // 2)]
    return [x * (1 - s) + x / factor * s for x, s in zip(f, (min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(n_rot // 2)))]


@pytest.mark.parametrize("n_rot,base,factor,orig,hi", [(128, 1e4, 4.0, 131072, 70), (64, 1e4, 8.0, 65536, 33), (128, 1e4, 4.0, 65536, 65), (64, 1e4, 4.0, 131072, 35), (64, 1e4, 4.0, 32768, 30),
                                                       (32, 100.0, 2.0, 200000, 31)])
def test_a_ramp_whose_slow_end_lies_behind_the_last_pair(n_rot, base, factor, orig, hi):
    """hi: the slow end, worked out by hand; the bounds are those of test_turns"""
    assert min(math.ceil(n_rot / 2 * math.log(orig / (2 * math.pi)) / math.log(base)), n_rot - 1) == hi
    r = q4gpu.Rope(n_rot, base, scaling="ramp", factor=factor, orig=orig, fast=32.0, slow=1.0)
    for i, f in enumerate(ramp(n_rot, base, factor, orig, 32.0, 1.0)):
        off = (Fraction(r.turn[i], 2**64) - Fraction(f) / TWO_PI) % 1
        assert min(off, 1 - off) <= Fraction(f) / 2**49 + Fraction(1, 2**52), i
