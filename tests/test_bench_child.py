"""`python bench.py --gpus N` runs its launcher as a child process: the process that counted the devices is never replaced by another
program (no exec), hands the launcher's status on and passes SIGTERM to it."""
import json
import os
import signal
import subprocess
import sys
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NO_EXEC = """
import os, sys
def refuse(*a, **k):
    raise AssertionError("exec from the benchmark's process")
for name in [n for n in dir(os) if n.startswith("exec")]:
    setattr(os, name, refuse)
sys.path.insert(0, {root!r})
import bench
bench._relaunch_one_rank_per_gpu(2, {script!r}, need_gpus=False)
"""


def _start(script, *argv):
    env = {k: v for k, v in os.environ.items() if k not in ("RANK", "LOCAL_RANK", "WORLD_SIZE", "MASTER_ADDR", "MASTER_PORT")}
    return subprocess.Popen([sys.executable, "-c", NO_EXEC.format(root=ROOT, script=str(script)), *argv], cwd=ROOT, env=env,
                            stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)


def test_the_launcher_is_a_child_and_prints_the_line():
    p = _start(os.path.join(ROOT, "tests", "bench_stub.py"), "--gpus", "2", "--steps", "2", "--warmup", "0", "--settle", "0")
    out, err = p.communicate(timeout=240)
    assert p.returncode == 0, err[-2000:]
    assert json.loads([l for l in out.splitlines() if l.startswith("{")][0])["n_gpus"] == 2


def test_a_failing_rank_fails_the_command(tmp_path):
    script = tmp_path / "fails.py"
    script.write_text("import os, sys; sys.exit(3 if os.environ['RANK'] == '1' else 0)\n")
    p = _start(script)
    _, err = p.communicate(timeout=240)
    assert p.returncode == 1, err[-2000:]                            # torch.distributed.run's status for a failed rank


@pytest.mark.parametrize("sig", [signal.SIGTERM, signal.SIGHUP])
def test_a_signal_reaches_the_ranks(tmp_path, sig):
    script = tmp_path / "sleeps.py"
    script.write_text(f"import os, time\nopen(os.path.join({str(tmp_path)!r}, 'pid' + os.environ['RANK']), 'w').write(str(os.getpid()))\ntime.sleep(120)\n")
    p = _start(script)
    pids = []
    try:
        end = time.time() + 100
        while len(pids) < 2 and time.time() < end and p.poll() is None:
            time.sleep(0.1)
            pids = [int(t) for r in "01" if (tmp_path / ("pid" + r)).exists() and (t := (tmp_path / ("pid" + r)).read_text())]
        assert len(pids) == 2
        p.send_signal(sig)
        _, err = p.communicate(timeout=90)
        assert p.returncode != 0, err[-2000:]
        end = time.time() + 20
        while time.time() < end and any(os.path.exists(f"/proc/{pid}") for pid in pids):
            time.sleep(0.1)
        assert not any(os.path.exists(f"/proc/{pid}") for pid in pids)
    finally:
        for pid in pids:
            try:                                                     # (a failed test only; never a process that has taken the number since)
                if str(script).encode() in open(f"/proc/{pid}/cmdline", "rb").read():
                    os.kill(pid, signal.SIGKILL)
            except (FileNotFoundError, ProcessLookupError):
                pass
        if p.poll() is None:
            p.kill()
