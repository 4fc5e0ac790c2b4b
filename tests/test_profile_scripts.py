"""The measuring scripts stop at the first step that fails (CPU: stand-ins for rocprofv3 and python3 that only write down that they
were called)."""
import os
import re
import shutil
import subprocess
import sys

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


# every script that starts something on the GPU; the stand-ins count those steps and fail the one that is asked for
ALL = sorted(f[:-3] for f in os.listdir(os.path.join(ROOT, "tools")) if f.endswith(".sh"))
ARGS = {"r5_occ": ["a=1", "b=2"], "r6_stats": ["name"]}                # what the others take has a default
STAND_IN = r"""#!/bin/bash
me=$(basename "$0"); d=.; j=; prev=
for a in "$@"; do [ "$prev" = -d ] && d=$a; [ "$prev" = --json ] && j=$a; prev=$a; done
case "$me $*" in
  "rocprofv3 "*|*bench.py*|*_stress.py*|*stress_parity.py*|*"-m pytest"*|*e2e_host_time.py*|*"ubench.py run"*) ;;
  *) [ -n "$j" ] && echo "{}" > "$j"; [ "$1" = -c ] && cat > /dev/null; echo "k_ksw_pair avg 1 us 1 %"; exit 0;;
esac
echo "$me $*" >> "$CALLS"
[ "$(wc -l < "$CALLS")" = "$FAIL_AT" ] && exit "$STATUS"
if [ "$me" = rocprofv3 ]; then mkdir -p "$d"; echo k_ksw_pair,k_prepack > "$d/1_kernel_stats.csv"; cp "$d/1_kernel_stats.csv" "$d/1_kernel_trace.csv"; fi
echo '{"metric k_ksw_pair'
"""


def _steps(tmp_path, script, fail_at, status):
    """(exit status, GPU steps started) of the script when its `fail_at`-th GPU step ends with `status`."""
    (tmp_path / "tools").mkdir()
    for s in ALL:
        shutil.copy(os.path.join(ROOT, "tools", s + ".sh"), tmp_path / "tools")
    lib, bin_, log = tmp_path / "indelope_amd" / "lib", tmp_path / "bin", tmp_path / "calls"
    lib.mkdir(parents=True)
    for so in ("libindelope_hip", "ab_one", "ab_two"):
        (lib / (so + ".so")).write_text(so)
    bin_.mkdir()
    log.write_text("")
    for name in ("rocprofv3", "python3", "python"):
        (bin_ / name).write_text(STAND_IN)
        (bin_ / name).chmod(0o755)
    env = dict(os.environ, PATH="%s:%s" % (bin_, os.environ["PATH"]), CALLS=str(log), FAIL_AT=str(fail_at), STATUS=str(status))
    r = subprocess.run(["bash", str(tmp_path / "tools" / (script + ".sh"))] + ARGS.get(script, []), env=env, stdin=subprocess.DEVNULL, capture_output=True,
                       timeout=100)
    assert (lib / "libindelope_hip.so").read_text() == "libindelope_hip"
    return r.returncode, log.read_text().splitlines()


@pytest.mark.parametrize("script", ALL)
def test_no_script_goes_on_after_a_failed_step(tmp_path, script):
    rc, steps = _steps(tmp_path, script, 0, 0)
    n = len(steps)
    assert n and rc == 0
    for i in sorted({1, 2, 3, n} & set(range(1, n + 1))):
        (tmp_path / str(i)).mkdir()
        rc, steps = _steps(tmp_path / str(i), script, i, 139)
        assert rc != 0 and len(steps) == i, (i, rc, steps)


@pytest.mark.parametrize("script", ALL)
def test_every_step_of_every_script_has_a_limit_that_kills(script):
    """`timeout` without -k leaves a process that ignores the first signal; rocprofv3 does after some errors."""
    with open(os.path.join(ROOT, "tools", script + ".sh")) as f:
        code = "".join(ln for ln in f if not ln.lstrip().startswith(("#", '"')))
    assert not re.search(r"timeout (?!-k 10 )", code)
    steps = [m.start() for m in re.finditer(r"(?<!-- )(?:rocprofv3 --\w|python3? (?:bench\.py|-m pytest|tools/\w*stress\w*\.py))", code)]
    for i in steps:
        assert re.search(r"(?:\$T |timeout -k 10 \d+ |^run \w+ )$", code[:i], flags=re.M), code[i:i + 60]
    assert steps


@pytest.mark.parametrize("script,shown", [("r6_stats", "5.25 {}"), ("r5_kstats", "5.25 7.5")])
def test_the_bench_line_is_found_before_the_profilers_last_words(tmp_path, script, shown):
    (tmp_path / "tools").mkdir()
    shutil.copy(os.path.join(ROOT, "tools", script + ".sh"), tmp_path / "tools")
    bin_ = tmp_path / "bin"
    bin_.mkdir()
    (bin_ / "rocprofv3").write_text("""#!/bin/bash
while [ "$1" != -d ]; do shift; done
mkdir -p "$2"; echo Name > "$2/1_kernel_stats.csv"
echo '{"metric": "m", "value": 5.25, "ms_per_step": 7.5, "kernel_ms": {}}'
echo "the profiler's last words"
""")
    (bin_ / "python3").write_text('#!/bin/bash\n[ "$1" != -c ] || exec %s "$@"\n' % sys.executable)
    for f in bin_.iterdir():
        f.chmod(0o755)
    r = subprocess.run(["bash", str(tmp_path / "tools" / (script + ".sh")), "steady"], stdin=subprocess.DEVNULL, capture_output=True, text=True, timeout=100,
                       env=dict(os.environ, PATH="%s:%s" % (bin_, os.environ["PATH"])))
    assert r.returncode == 0 and shown in r.stdout, (r.stdout, r.stderr)
