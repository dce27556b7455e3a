"""bench.py under somebody else's launcher: a rung whose guard fires is gone before the next one starts, exactly one line is printed,
and no rung outlives the rank's process (CPU: the rungs are small scripts on bench.py's own guards)."""
import os
import signal
import subprocess
import sys
import time

import pytest

from conftest import REPO

_RUNG = r'''
import os, sys, time
sys.path.insert(0, %(repo)r)
import bench
log = open(os.environ["RUNG_LOG"], "a")
attempt = int(os.environ.get("DSW_PG_ATTEMPT", "0"))
earlier = [int(ln.split()[0]) for ln in open(os.environ["RUNG_LOG"])]
alive = [p for p in earlier if os.path.exists("/proc/%%d" %% p)]
print(os.getpid(), attempt, len(alive), os.environ.get("DSW_BENCH_COLLECTIVES"), os.environ.get("DSW_BENCH_NO_GRAPH"), file=log, flush=True)
bench._die_with_supervisor()
assert "DSW_BENCH_SUPERVISOR" not in os.environ
%(body)s
'''


def _start(tmp_path, body, **env):
    script = tmp_path / "rung.py"
    script.write_text(_RUNG % {"repo": REPO, "body": body})
    (tmp_path / "log").write_text("")
    code = "import sys; sys.path.insert(0, %r); import bench; sys.exit(bench.supervise([sys.executable, %r]))" % (REPO, str(script))
    clean = {k: v for k, v in os.environ.items() if not k.startswith("DSW_")}
    return subprocess.Popen([sys.executable, "-c", code], env=dict(clean, RUNG_LOG=str(tmp_path / "log"), **env), stdout=subprocess.PIPE,
                            stderr=subprocess.PIPE, text=True)


def _log(tmp_path):
    return [ln.split() for ln in (tmp_path / "log").read_text().splitlines()]


def test_two_guards_and_a_late_main_thread(tmp_path):
    """Both timers of a rung are due and its main thread comes back: one hand-over, one line, the line's exit code."""
    p = _start(tmp_path, '''
if attempt == 0:
    bench._arm_watchdog(0, 2, 0.3, "the first replay", retry=True)
    bench._arm_watchdog(0, 2, 0.3, "the run", retry=True)
    time.sleep(3)
bench.print_line({"metric": "m", "attempt": attempt})
''')
    out, err = p.communicate(timeout=120)
    assert p.returncode == 0, err[-2000:]
    assert out.splitlines() == ['{"metric": "m", "attempt": 1}'] and err.count("re-executing") == 1
    assert [r[1:] for r in _log(tmp_path)] == [["0", "0", "None", "None"], ["1", "0", "eager", "None"]]


def test_a_line_that_is_out_is_not_measured_again(tmp_path):
    p = _start(tmp_path, '''
bench._arm_watchdog(0, 2, 0.5, "the run", retry=True)
bench.print_line({"metric": "m"})
time.sleep(60)
''')
    out, err = p.communicate(timeout=120)
    assert p.returncode == 124 and out.splitlines() == ['{"metric": "m"}'] and "giving up" in err and len(_log(tmp_path)) == 1


def test_the_ladder_ends(tmp_path):
    p = _start(tmp_path, 'bench._arm_watchdog(0, 2, 0.2, "the run", retry=True); time.sleep(60)')
    out, err = p.communicate(timeout=120)
    assert p.returncode == 124 and out == ""
    assert [r[1:] for r in _log(tmp_path)] == [["0", "0", "None", "None"], ["1", "0", "eager", "None"], ["2", "0", "eager", "1"]]


@pytest.mark.parametrize("body,code", [("sys.exit(3)", 3), ("os.kill(os.getpid(), 9)", 137)])
def test_a_rung_that_fails_is_the_ranks_failure(tmp_path, body, code):
    p = _start(tmp_path, body)
    p.communicate(timeout=120)
    assert p.returncode == code and len(_log(tmp_path)) == 1


def test_a_rung_that_cannot_end_itself_is_killed(tmp_path):
    """No guard of its own: the supervisor's limit (its run limit and a minute: 24 s here) ends it."""
    p = _start(tmp_path, "time.sleep(600) if attempt == 0 else bench.print_line({'metric': 'm'})", DSW_BENCH_TIMEOUT="-40")
    out, err = p.communicate(timeout=120)
    assert p.returncode == 0 and out.splitlines() == ['{"metric": "m"}'], err[-1500:]
    assert [r[1:3] for r in _log(tmp_path)] == [["0", "0"], ["1", "0"]]


@pytest.mark.parametrize("sig", [signal.SIGTERM, signal.SIGKILL])
def test_a_rung_does_not_outlive_its_rank(tmp_path, sig):
    p = _start(tmp_path, "open(os.environ['RUNG_LOG'] + '.ready', 'w').close(); time.sleep(600)")
    end = time.time() + 60
    while not (tmp_path / "log.ready").exists() and time.time() < end:
        time.sleep(0.05)
    pid = int(_log(tmp_path)[0][0])
    p.send_signal(sig)
    p.communicate(timeout=60)
    assert p.returncode == (128 + sig if sig == signal.SIGTERM else -sig)
    end = time.time() + 20
    while os.path.exists("/proc/%d" % pid) and time.time() < end:
        if open("/proc/%d/stat" % pid).read().rsplit(")", 1)[1].split()[0] == "Z":         # (an orphan that nobody has waited for)
            return
        time.sleep(0.05)
    assert not os.path.exists("/proc/%d" % pid)
