"""What no setting, script or source file may reach, checked on the sources and the built libraries (no device needed)."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tracked(*suffixes):
    """Files under version control with one of these suffixes (the working tree's own files where there is no git: an exported copy)."""
    try:
        names = subprocess.run(["git", "ls-files"], cwd=ROOT, capture_output=True, text=True, check=True).stdout.splitlines()
    except (OSError, subprocess.CalledProcessError):
        names = [os.path.relpath(os.path.join(d, f), ROOT) for d, _, fs in os.walk(ROOT) for f in fs]
    return [n for n in names if n.endswith(suffixes) and os.path.exists(os.path.join(ROOT, n))]


def _read(name):
    with open(os.path.join(ROOT, name), "rb") as f:
        return f.read()


# ---- the pair kernel's claim order (scan_teddy_pair.hip): one counter.  With several, a workgroup that takes from another's counter once its
# own is exhausted can draw a group in front of one it has not resolved; its look-back then waits for itself and only the spin limit ends it.

@pytest.mark.parametrize("lib", ["libcoregex_hip.so", "libcoregex_hip_rocm.so"])
def test_no_setting_of_the_library_spreads_the_group_claims(lib):
    path = os.path.join("coregex_amd", lib)
    if not os.path.exists(os.path.join(ROOT, path)):
        pytest.skip(f"{lib} is not built")
    assert b"CXG_PAIR_NCTR" not in _read(path)


def test_no_script_or_document_offers_several_group_counters():
    here = os.path.relpath(os.path.abspath(__file__), ROOT)
    names = [n for n in _tracked(".hip", ".h", ".hpp", ".cc", ".py", ".sh") if n != here] + ["README.md"]
    offers = [n for n in names if re.search(rb"PAIR_NCTR|pair_nctr\b", _read(n))]
    assert offers == []


# ---- device code writes through vector stores only: nothing goes through the scalar data cache (its stores, atomics, write-back, discard)

def test_no_source_writes_through_the_scalar_data_cache():
    names = _tracked(".hip", ".cc", ".cpp", ".h", ".hpp", ".c", ".s", ".S", ".py", ".sh", "Makefile")
    scalar_write = re.compile(rb"\bs_(?:buffer_|scratch_)?(?:store|atomic)_\w+|\bs_dcache_(?:wb|discard)\w*")
    assert len(names) > 100
    assert [(n, m.group().decode()) for n in names for m in [scalar_write.search(_read(n))] if m] == []


# ---- no setting of the library leaves out part of a scan

@pytest.mark.parametrize("lib", ["libcoregex_hip.so", "libcoregex_hip_rocm.so"])
def test_no_setting_of_the_library_skips_work(lib):
    path = os.path.join("coregex_amd", lib)
    if not os.path.exists(os.path.join(ROOT, path)):
        pytest.skip(f"{lib} is not built")
    assert b"CXG_DEBUG" not in _read(path)                           # (it skipped the lane walk or the look-back and returned wrong rows)


def test_the_benchmark_checks_its_rows_whatever_the_environment_says():
    assert b"CXG_DEBUG" not in _read("bench.py")
