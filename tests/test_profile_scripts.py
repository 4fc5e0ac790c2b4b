"""The measuring scripts stop at the first step that fails (CPU: stand-ins for rocprofv3 and python3 that only write down that they
were called)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCRIPTS = ["profile_round", "pmc_mix", "r4_fb", "r4_prepack", "r4_kpmc", "r5_occ"]


def _run(tmp_path, script, rocprof_status, python_status):
    """(exit status, calls) of the script in a tree of its own."""
    (tmp_path / "tools").mkdir()
    for s in SCRIPTS:
        shutil.copy(os.path.join(ROOT, "tools", s + ".sh"), tmp_path / "tools")
    bin_, log = tmp_path / "bin", tmp_path / "calls"
    bin_.mkdir()
    for name, status in (("rocprofv3", rocprof_status), ("python3", python_status)):
        (bin_ / name).write_text('#!/bin/bash\necho "%s $*" >> %s\necho "{}"\nexit %d\n' % (name, log, status))
        (bin_ / name).chmod(0o755)
    env = dict(os.environ, PATH="%s:%s" % (bin_, os.environ["PATH"]))
    r = subprocess.run(["bash", str(tmp_path / "tools" / (script + ".sh")), "a=1", "b=2"], env=env, capture_output=True, timeout=60)
    return r.returncode, log.read_text().splitlines()


@pytest.mark.parametrize("script", SCRIPTS)
@pytest.mark.parametrize("status", [124, 134, 139])
def test_nothing_runs_behind_a_failed_profile(tmp_path, script, status):
    rc, calls = _run(tmp_path, script, status, 0)
    assert rc == status
    assert [c.startswith("rocprofv3") for c in calls].index(True) == len(calls) - 1, calls


@pytest.mark.parametrize("script", ["profile_round", "r4_fb"])
def test_nothing_runs_behind_a_failed_program(tmp_path, script):
    rc, calls = _run(tmp_path, script, 0, 134)
    assert rc != 0 and len(calls) == 1, calls


@pytest.mark.parametrize("script", SCRIPTS)
def test_every_step_on_the_gpu_has_a_limit(script):
    with open(os.path.join(ROOT, "tools", script + ".sh")) as f:
        code = "".join(ln for ln in f if not ln.lstrip().startswith(("#", '"')))
    assert 'T="timeout -k 10 ' in code
    steps = [m.start() for m in re.finditer(r"(?<!-- )(?:rocprofv3 --\w|python3 bench\.py)", code)]
    assert steps and all(code[:i].endswith("$T ") for i in steps)
