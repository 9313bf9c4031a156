"""The table-walking DFA-pair kernel's read budget (scan_dfa.h kSerialReads, kSerialLimit) on its CPU twin.

A program whose every search runs to the end of a stretch without synchronising bytes walks matches x stretch bytes.  The kernel counts the
bytes a lane reads beyond its staged window; past the budget it raises kErrSerialLimit (the call ends in CXG_E_INPUT) and reads no more."""
import os
import re

import numpy as np
import pytest

import coregex_amd as cx
import emu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
QUADRATIC = r"\D+?xyzabcx|bcxy|cxyz|xyza[a-c]"
E_SERIAL_LIMIT = -32


def _constant(name):
    src = open(os.path.join(ROOT, "coregex_amd", "csrc", "device", "scan_dfa.h")).read()
    return eval(re.search(rf"constexpr \w+ {name} = ([0-9u<* ]+);", src).group(1).replace("u", ""))


def _periodic(n):
    return np.frombuffer(b"abcxyza:c" * n, dtype=np.uint8)


@pytest.mark.parametrize("n", [0, 1, 50, 500, 1800])
def test_below_the_budget_the_rows_are_the_oracles(oracle, n):
    hay = _periodic(n)
    got, reads = emu.find_all_budget(cx.compile(QUADRATIC).blob(), hay)
    assert np.array_equal(got, oracle.Regex(QUADRATIC).find_all_index(hay))
    assert reads <= _constant("kSerialReads")


def test_a_quadratic_walk_is_refused_after_its_budget():
    got, reads = emu.find_all_budget(cx.compile(QUADRATIC).blob(), _periodic(9000))
    assert got == E_SERIAL_LIMIT
    assert reads == _constant("kSerialReads")                        # spent, and not a byte more


def test_one_walk_past_the_cut_is_refused():
    """A single search that is still running kSerialLimit bytes behind the window: linear, so the cut refuses it and not the read count."""
    hay = np.frombuffer(b"x" * (2 * _constant("kSerialLimit")), dtype=np.uint8)
    got, reads = emu.find_all_budget(cx.compile(r"\D+?xyzabcx|bcxy").blob(), hay)
    assert got == E_SERIAL_LIMIT and reads <= _constant("kSerialReads")


def test_no_script_sends_the_quadratic_program_to_the_device():
    scripts = os.path.join(ROOT, "scripts")
    holds = [f for f in os.listdir(scripts) if f.endswith((".py", ".sh")) and "xyzabcx" in open(os.path.join(scripts, f)).read()]
    assert holds == ["gpu_fuzz.py"]                                  # whose random patterns reach it (FUZZ_WIDE, seed 82): left out there
    src = open(os.path.join(scripts, "gpu_fuzz.py")).read()
    assert src.count("xyzabcx") == 1 and f'LEFT_OUT = {{r"{QUADRATIC}"}}' in src
    loop = src[src.index("while len(seen) < npat:"):]
    assert loop.index("if pat in LEFT_OUT:") < loop.index("cx.compile(pat)")
