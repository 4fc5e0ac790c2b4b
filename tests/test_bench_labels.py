"""What bench.py says its CPU side is (CPU only: the oracle stands in for the device)."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


@pytest.mark.parametrize("compiled", [True, False])
def test_the_break_even_says_which_ksw2_it_is_up_against(oracle, monkeypatch, compiled):
    """Where the reference's ksw2 is not built the CPU side runs the scalar restatement, which is slower."""
    import bench
    monkeypatch.setattr(type(oracle), "use_reference_ksw", lambda self, on: compiled and on)
    out = bench.break_even(oracle, sizes=(1,), reps=1)
    assert ("reference ksw2_extz2_sse.c compiled" in out["workload"]) == compiled
    assert ("scalar restatement" in out["workload"]) == (not compiled)
    assert [r["regions"] for r in out["rows"]] == [1]
