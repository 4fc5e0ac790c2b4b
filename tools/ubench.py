#!/usr/bin/env python3
"""Builds and runs the microbenchmarks tools/ubench_*.hip.

A binary carries the hash of the source and flags it was built from in its name (tools/ubench_ksw.<sha16>.bin), so what runs is
always what stands in the tree: an older binary is not found.  Build where hipcc is, run where the GPU is.
usage: tools/ubench.py build                    all of them; binaries of earlier sources are removed
       tools/ubench.py check                    exit 2 and say which one is missing, unless all are built
       tools/ubench.py run NAME LOG [SECONDS]   e.g. `run ksw out/ubench_ksw.txt`: LOG is written only when the run succeeds,
                                                its first line names the source and its hash (limit: 120 s unless given)"""
import glob
import hashlib
import os
import subprocess
import sys

TOOLS = os.path.dirname(os.path.abspath(__file__))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# (the host pass warns that it does not know the feature: harmless)
FLAGS = ["--offload-arch=gfx950", "-O3", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def source(name):
    return os.path.join(TOOLS, "ubench_%s.hip" % name)


def names():
    return sorted(os.path.basename(p)[len("ubench_"):-len(".hip")] for p in glob.glob(os.path.join(TOOLS, "ubench_*.hip")))


def sha16(name):
    h = hashlib.sha256(" ".join(FLAGS).encode())
    with open(source(name), "rb") as f:
        h.update(f.read())
    return h.hexdigest()[:16]


def binary(name):
    return os.path.join(TOOLS, "ubench_%s.%s.bin" % (name, sha16(name)))


def build():
    for n in names():
        exe = binary(n)
        subprocess.check_call([HIPCC] + FLAGS + ["-o", exe, source(n)])
        for old in glob.glob(os.path.join(TOOLS, "ubench_%s.bin" % n)) + glob.glob(os.path.join(TOOLS, "ubench_%s.*.bin" % n)):
            if old != exe:
                os.remove(old)
        print(exe)
    return 0


def missing(which):
    lost = [n for n in which if not os.path.exists(source(n)) or not os.path.exists(binary(n))]
    for n in lost:
        print("ubench: tools/ubench_%s.hip is not built as it stands (tools/ubench.py build)" % n, file=sys.stderr)
    return lost


def run(name, log, limit):
    if missing([name]):
        return 2
    try:
        r = subprocess.run([binary(name)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=limit)
    except subprocess.TimeoutExpired:
        print("ubench: %s ran into its limit of %g s" % (name, limit), file=sys.stderr)
        return 124
    if r.returncode:
        print("ubench: %s ended with status %d\n%s" % (name, r.returncode, r.stdout[-2000:]), file=sys.stderr)
        return r.returncode if r.returncode > 0 else 128 - r.returncode
    with open(log, "w") as f:
        f.write("tools/ubench_%s.hip sha16 %s (hipcc %s)\n%s" % (name, sha16(name), " ".join(FLAGS), r.stdout))
    return 0


def main(argv):
    if argv == ["build"]:
        return build()
    if argv == ["check"]:
        return 2 if missing(names()) else 0
    if len(argv) in (3, 4) and argv[0] == "run":
        return run(argv[1], argv[2], float(argv[3]) if len(argv) == 4 else 120.0)
    print(__doc__, file=sys.stderr)
    return 2


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
