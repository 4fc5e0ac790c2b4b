"""What the sources of GPU code may not hold, comments included (CPU only: text of the tree, nothing is run)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SKIP = {".git", "_work", "gpurun_out", "__pycache__", ".pytest_cache", ".hypothesis", "build", "profiles"}
EXT = (".hip", ".h", ".hpp", ".c", ".cpp", ".s", ".S", ".py", ".sh", ".nim", ".mk")


def _sources():
    for d, dirs, files in os.walk(ROOT):
        dirs[:] = sorted(x for x in dirs if x not in SKIP)
        for f in sorted(files):
            if f.endswith(EXT) or f == "Makefile":
                yield os.path.join(d, f)


def _hits(pattern):
    rx, out = re.compile(pattern), []
    for path in _sources():
        with open(path, errors="replace") as fh:
            out += ["%s:%d: %s" % (os.path.relpath(path, ROOT), n, m.group(0)) for n, ln in enumerate(fh, 1) for m in rx.finditer(ln)]
    return out


def test_the_walk_sees_the_kernels():
    seen = {os.path.relpath(p, ROOT) for p in _sources()}
    assert {"indelope_amd/csrc/kernels.h", "indelope_amd/csrc/indelope_hip.hip", "tools/ubench_ksw.hip", "tools/ubench_issue.hip"} <= seen


def test_nothing_writes_through_the_scalar_data_cache():
    """Scalar memory stores and atomics, and that cache's write-back and discard: results leave by vector stores only."""
    assert _hits(r"(?<![A-Za-z0-9])s_(?:[a-z]+_)?(?:store|atomic)[a-z0-9_]*|(?<![A-Za-z0-9])s_dcache_(?:wb|discard)[a-z_]*") == []


def test_no_packed_fp32():
    """v_pk_{add,mul,fma}_f32 have given wrong results on gfx950 with no error, in ways that tests do not reliably show."""
    assert _hits(r"v_pk_(?:add|mul|fma)_f32") == []
