"""How the libraries are built: the compiler's flags of every HIP object (make's own dry run), and what build() compiles."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "coregex_amd", "csrc")


def test_every_hip_object_is_compiled_without_packed_fp32():
    lines = subprocess.run(["make", "-n", "-B", "-C", CSRC, "all"], capture_output=True, text=True, check=True).stdout.splitlines()
    compiles = [l for l in lines if "-x hip" in l and " -c " in l]
    assert len(compiles) >= 20 and all("--offload-arch=gfx950" in l for l in compiles)
    assert all("-Xclang -target-feature -Xclang -packed-fp32-ops" in l for l in compiles)


def test_build_compiles_everything_on_every_call(monkeypatch):
    sys.path.insert(0, ROOT)
    import __graft_entry__ as entry
    ran = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, *a, **k: ran.append(cmd))
    entry.build()
    made = {os.path.relpath(c[c.index("-C") + 1], ROOT): c for c in ran if c[0] == "make"}
    assert set(made) == {os.path.join("coregex_amd", "csrc"), "oracle", os.path.join("tests", "emu")}
    assert all("-B" in c for c in made.values())                     # ... whatever is built already
