"""indelope_amd/build.py: what the compiler is called with, and when (CPU: the compilers are not run)."""
import os
import re
import shutil
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from indelope_amd import build as B  # noqa: E402


@pytest.fixture
def calls(tmp_path, monkeypatch):
    """The commands of a build into an empty directory; the "compilers" only leave their output file behind."""
    seen = []

    def call(cmd, **kw):
        seen.append(list(cmd))
        if "-o" in cmd:
            with open(cmd[cmd.index("-o") + 1], "w") as f:
                f.write("built %d" % len(seen))
    monkeypatch.setattr(B.subprocess, "check_call", call)
    monkeypatch.setattr(B, "LIBDIR", str(tmp_path / "lib"))
    return seen


def test_the_library_is_built_without_packed_fp32(calls):
    lib, _ = B.build()
    hip = [c for c in calls if lib in c]
    assert len(hip) == 1 and hip[0][0] == B.HIPCC
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in " ".join(hip[0])
    assert "--offload-arch=gfx950" in hip[0] and "-ffp-contract=off" in hip[0]


def test_the_evidence_is_of_the_build(monkeypatch):
    """Counters taken from other flags are of another build; the tools that compile the kernels for a report take the library's flags."""
    import bench
    sha = bench.src_sha16()
    monkeypatch.setattr(B, "HIPFLAGS", B.HIPFLAGS + ["-O2"])
    assert bench.src_sha16() != sha
    for f in ("tools/spill_report.py", "tools/profile_round.sh"):
        text = open(os.path.join(ROOT, f)).read()
        assert "HIPFLAGS" in text and not re.search(r"offload-arch|ffp-contract|/hipcc", text), f


def test_a_change_of_the_flags_builds_again(calls, monkeypatch):
    lib, _ = B.build()
    n = len(calls)
    B.build()
    assert len(calls) == n                                       # nothing to do
    t = os.path.getmtime(B.__file__) - 10
    os.utime(lib, (t, t))
    mtime = os.path.getmtime
    monkeypatch.setattr(B.os.path, "getmtime", lambda p: t - 10 if p.endswith((".hip", ".h")) else mtime(p))
    B.build()
    assert len(calls) == n + 1 and lib in calls[-1]


def test_the_build_entry_compiles_what_is_there_too(calls):
    import __graft_entry__
    __graft_entry__.build()
    first = [c for c in calls if c[0] in ("g++", B.HIPCC)]
    del calls[:]
    __graft_entry__.build()
    assert len(first) == 2 and [c for c in calls if c[0] in ("g++", B.HIPCC)] == first


@pytest.fixture
def sources(tmp_path, monkeypatch):
    """bench.py on a copy of the library's sources."""
    import bench
    for d in (("indelope_amd", "csrc"), ("include",)):
        shutil.copytree(os.path.join(ROOT, *d), str(tmp_path.joinpath(*d)))
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    return bench, tmp_path / "indelope_amd" / "csrc"


def test_a_comment_makes_no_other_build(sources):
    """A changed comment left the committed counters marked as another build's."""
    bench, csrc = sources
    sha = bench.src_sha16()
    f = csrc / "kernels.h"
    text = f.read_text()
    f.write_text("// a remark\n/* and one\n   of 2 lines */\n" + text.replace(";\n", ";   // \"quoted\" and it's fine\n\n", 50))
    assert bench.src_sha16() == sha
    f.write_text(text + "\n__device__ int one_more;\n")
    assert bench.src_sha16() != sha


@pytest.mark.parametrize("a,b", [
    ('x = "a // b";', 'x = "a // c";'), ('x = "a  b";', 'x = "a b";'), ("x = '\"'; y = 1; // '", "x = '\"'; y = 2; // '"),
    ("x = 0x49'4c; y = 1;", "x = 0x49'4c; y = 2;"), ('x = "\\"/*"; y = 1; /**/', 'x = "\\"/*"; y = 2; /**/'),
    ("#define A 1\nB", "#define A 1 B"), ("a /* c */ b", "ab"), ("x = '/'; y = 1;", "x = '/'; y = 2;")])
def test_a_change_of_code_makes_another_build(a, b):
    import bench
    assert bench._code(a) != bench._code(b)


@pytest.mark.parametrize("a,b", [
    ("x = 1; // one", "x = 1;"), ("x = 1;\n// one\ny = 2;", "x = 1;\n\ty = 2;  /* two */\n"), ("x = 'a'; // 'b", "x = 'a';"),
    ('x = "a"; /* " */ y = 1;', 'x = "a"; y = 1;')])
def test_what_is_no_code(a, b):
    import bench
    assert bench._code(a) == bench._code(b)
