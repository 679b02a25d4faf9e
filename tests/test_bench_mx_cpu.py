"""bench.py's ``--mx`` without a GPU: which workloads take it, and that the record says so."""

import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import bench

ROOT = Path(__file__).resolve().parents[1]


def test_workloads_without_projections_refuse_it():
    p = subprocess.run([sys.executable, str(ROOT / "bench.py"), "--mx"], capture_output=True, text=True, timeout=120,
                       cwd=ROOT)
    assert p.returncode == 2 and "has no projections" in p.stderr


def test_records_name_the_weights():
    plain, mx = SimpleNamespace(mx=False), SimpleNamespace(mx=True)
    assert bench._step_dtype(plain) == "bf16" and bench._mx_words(plain) == ""
    assert "mxfp4" in bench._step_dtype(mx) and "4-bit weights" in bench._mx_words(mx)
