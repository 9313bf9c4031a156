"""How the libraries are built: the compiler's flags of every HIP object (make's own dry run)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "coregex_amd", "csrc")


def test_every_hip_object_is_compiled_without_packed_fp32():
    lines = subprocess.run(["make", "-n", "-B", "-C", CSRC, "all"], capture_output=True, text=True, check=True).stdout.splitlines()
    compiles = [l for l in lines if "-x hip" in l and " -c " in l]
    assert len(compiles) >= 20 and all("--offload-arch=gfx950" in l for l in compiles)
    assert all("-Xclang -target-feature -Xclang -packed-fp32-ops" in l for l in compiles)
