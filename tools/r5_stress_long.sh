cd "$(dirname "$0")/.." || exit 1
set -eo pipefail                             # a step that failed, faulted or ran into its limit ends the script: nothing more is started on the GPU
mkdir -p gpurun_out/stress
S=${1:-201}
run() { name=$1; rc=0; shift; timeout -k 10 2400 "$@" > gpurun_out/stress/$name.txt 2>&1 || rc=$?; echo "== $name rc=$rc : $(tail -1 gpurun_out/stress/$name.txt | cut -c1-200)"; grep -c DIFF gpurun_out/stress/$name.txt || true; return $rc; }
run pair_a python tools/ksw_pair_stress.py $S 700
run pair_b python tools/ksw_pair_stress.py $((S+1)) 700
run ksw python tools/ksw_stress.py $S 1000
run regions_params python tools/stress_parity.py 1200 $S params
run regions_lengths python tools/stress_parity.py 600 $((S+2)) lengths
run threads python tools/thread_stress.py 6 60 $S
run fb python tools/fb_stress.py $S 60
run contig python tools/contig_stress.py 15000 $S
run sweep python tools/sweep_stress.py 30 $S
python - <<PY
import sys
sys.path.insert(0, '.')
import bench
print("src_sha16", bench.src_sha16())
PY
