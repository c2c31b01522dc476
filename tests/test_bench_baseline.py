"""The CPU baseline of the bench line: left out only where the reference's kernels are not built."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import oracle as O

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bench  # noqa: E402

Q4K, Q80 = bench.TYPE_IDS["q4_K"], bench.TYPE_IDS["q8_0"]


def test_without_the_reference_kernels(monkeypatch):
    monkeypatch.setattr(O, "load_ref", lambda *a: None)
    monkeypatch.setattr(bench, "cpu_pass", lambda *a: pytest.fail("nothing to run"))
    r = bench.cpu_baseline({}, {}, [(4, Q80, 64, 256), (4, Q4K, 64, 256)], 0.1)
    assert r == {"unavailable": "the reference kernels (oracle/_ref) are not built"}


def test_a_failure_is_not_a_missing_baseline(monkeypatch):
    """A broken build, or a RuntimeError of torch or CUDA in a pass, with the kernels there."""
    def broken(*a):
        raise RuntimeError("CUDA error")

    monkeypatch.setattr(O, "load_ref", lambda *a: object())
    monkeypatch.setattr(bench, "cpu_pass", broken)
    with pytest.raises(RuntimeError):
        bench.cpu_baseline({}, {}, [(4, Q4K, 64, 256)], 0.1)


def test_q8_0_needs_no_reference_kernels(monkeypatch):
    monkeypatch.setattr(O, "load_ref", lambda *a: None)
    w = O.quantize_rtn(O.Q8_0, np.ones((64, 256), np.float32)).reshape(64, -1)
    r = bench.cpu_baseline({(Q80, 64, 256): w}, {(4, 256): np.ones((4, 256), np.float32)},
                           [(4, Q80, 64, 256)], 0.01)
    assert r["kind"] == "port" and r["value"] > 0


@pytest.mark.skipif(O.load_ref() is not None, reason="the reference's kernels are built: its arm runs")
def test_the_reference_arm_without_its_kernels():
    """One JSON line on the standard output, as every run of the bench prints it."""
    r = subprocess.run([sys.executable, bench.__file__, "--impl", "reference", "--steps", "1", "--warmup", "0"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0
    line = json.loads(r.stdout)
    assert line["impl"] == "reference" and line["unavailable"]
