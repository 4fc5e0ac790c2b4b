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


# scalar instructions that set SCC (moves, multiplies, selects and branches do not)
_SETS_SCC = re.compile(r"(?<![A-Za-z0-9_])s_(?:and|or|xor|andn[12]|orn[12]|nand|nor|xnor|not|addc?|subb?|min|max|cmp|bitcmp[01]|lshl(?:[1-4]_add)?|"
                       r"lshr|ashr|bfe|abs|absdiff|bcnt[01]|wqm|quadmask)_[a-z0-9_]+")


def _asm_statements(text):
    """(line, statement) of every inline assembly statement: up to the parenthesis that closes it, strings skipped."""
    for m in re.finditer(r"(?<!\w)asm\s*(?:volatile\s*)?(?:goto\s*)?\(", text):
        i, depth, quoted = m.end(), 1, False
        while depth:
            c = text[i]
            quoted ^= c == '"' and text[i - 1] != "\\"
            depth += 0 if quoted else {"(": 1, ")": -1}.get(c, 0)
            i += 1
        yield text.count("\n", 0, m.start()) + 1, text[m.start():i]


def test_assembly_that_sets_scc_says_so():
    """The compiler keeps loop conditions in SCC: a statement that sets it without a clobber decides when the loop around it ends."""
    seen, lost = 0, []
    for path in _sources():
        if path.endswith((".h", ".hip")):
            with open(path, errors="replace") as f:
                for line, asm in _asm_statements(f.read()):
                    if _SETS_SCC.search(asm):
                        seen += 1
                        if '"scc"' not in asm:
                            lost.append("%s:%d" % (os.path.relpath(path, ROOT), line))
    assert seen >= 9 and lost == []
