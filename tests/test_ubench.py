"""tools/ubench.py: what runs is what stands in the tree, and a run that did not happen leaves no evidence (CPU: the "compiler"
is a script that wraps the source, the "benchmarks" are shell scripts)."""
import importlib.util
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def ub(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("ubench_under_test", os.path.join(ROOT, "tools", "ubench.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    cc = tmp_path / "cc"
    cc.write_text("#!/bin/bash\nwhile [ \"$1\" != -o ]; do shift; done\n(echo '#!/bin/bash'; cat \"$3\") > \"$2\"; chmod +x \"$2\"\n")
    cc.chmod(0o755)
    monkeypatch.setattr(m, "TOOLS", str(tmp_path))
    monkeypatch.setattr(m, "HIPCC", str(cc))
    (tmp_path / "ubench_a.hip").write_text("echo first\n")
    (tmp_path / "ubench_b.hip").write_text("echo b\n")
    return m


def test_a_run_names_its_source(ub, tmp_path):
    assert ub.main(["check"]) == 2
    assert ub.main(["build"]) == 0
    assert ub.main(["check"]) == 0
    log = tmp_path / "a.txt"
    assert ub.main(["run", "a", str(log)]) == 0
    head, body = log.read_text().split("\n", 1)
    assert head.startswith("tools/ubench_a.hip sha16 %s " % ub.sha16("a")) and body == "first\n"


def test_a_missing_binary_is_reported_and_leaves_no_log(ub, tmp_path, capsys):
    log = tmp_path / "a.txt"
    assert ub.main(["run", "a", str(log)]) == 2
    assert "ubench_a.hip is not built" in capsys.readouterr().err and not log.exists()
    assert ub.main(["run", "nosuch", str(log)]) == 2 and not log.exists()


def test_a_binary_of_an_earlier_source_is_not_run(ub, tmp_path):
    ub.main(["build"])
    old = ub.binary("a")
    (tmp_path / "ubench_a.bin").write_text("left by an earlier build step")
    (tmp_path / "ubench_a.hip").write_text("echo second\n")
    log = tmp_path / "a.txt"
    assert ub.main(["run", "a", str(log)]) == 2 and not log.exists()
    ub.main(["build"])
    assert not os.path.exists(old) and not (tmp_path / "ubench_a.bin").exists() and os.path.exists(ub.binary("b"))
    assert ub.main(["run", "a", str(log)]) == 0 and log.read_text().endswith("\nsecond\n")


@pytest.mark.parametrize("body,limit,rc", [("echo half; exit 3", "10", 3), ("exec sleep 30", "0.3", 124), ("kill -9 $$", "10", 137)])
def test_a_failed_run_gives_its_status_and_no_log(ub, tmp_path, body, limit, rc):
    (tmp_path / "ubench_a.hip").write_text(body + "\n")
    ub.main(["build"])
    log = tmp_path / "a.txt"
    assert ub.main(["run", "a", str(log), limit]) == rc and not log.exists()


def test_the_profile_script_starts_no_binary_by_itself():
    with open(os.path.join(ROOT, "tools", "profile_round.sh")) as f:
        lines = [ln.strip() for ln in f if "ubench" in ln and not ln.lstrip().startswith("#")]
    assert lines and all(re.match(r"python3 tools/ubench\.py (check|run \w+ \S+) \|\| exit", ln) for ln in lines), lines
