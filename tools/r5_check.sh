#!/bin/bash
# The GPU suite (or a subset), then a default bench line.
#   tools/r5_check.sh [pytest -k expression | all | none] [bench args...]
cd "$(dirname "$0")/.." || exit 1
set -eo pipefail                             # a step that failed, faulted or ran into its limit ends the script: nothing more is started on the GPU
mkdir -p gpurun_out
sel=${1:-all}; [ $# = 0 ] || shift
if [ "$sel" = all ]; then timeout -k 10 600 python -m pytest tests -m gpu -x -q > gpurun_out/r5_pytest.txt 2>&1
elif [ "$sel" != none ]; then timeout -k 10 600 python -m pytest tests -m gpu -x -q -k "$sel" > gpurun_out/r5_pytest.txt 2>&1; fi
[ "$sel" = none ] || tail -5 gpurun_out/r5_pytest.txt
t0=$(date +%s); timeout -k 10 600 python bench.py "$@" > gpurun_out/r5_bench.json 2> gpurun_out/r5_bench.err; echo "bench wall $(( $(date +%s) - t0 )) s"
grep -v amdgpu.ids gpurun_out/r5_bench.err | tail -5 || true
python - <<PY
import json
try:
    d=json.loads(open("gpurun_out/r5_bench.json").read().strip().splitlines()[-1])
    print(json.dumps(d["digest"]))
except Exception as e:
    print("bench failed", e)
PY
