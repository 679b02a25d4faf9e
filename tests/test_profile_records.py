"""The counters' records under profiles/ that bench.py reports: they count for the kernel sources that they were
collected on, and are dropped from its line with any others."""

import json
from pathlib import Path

import bench

PROFILES = Path(bench.__file__).resolve().parent / "profiles"


def test_records_are_of_these_sources():
    records = sorted(PROFILES.glob("attn_fwd_*.json"))
    assert records
    for f in records:
        assert json.loads(f.read_text())["source_sha"] == bench.kernel_source_hash(), (
            f"{f.name}: block_attn.hip or fm_device.h changed; collect the counters again, or keep what the attention "
            "does not use in another header")


def test_the_default_line_has_them():
    workload = "c3-qwen3-8b-paged-b64"
    assert bench.traffic_record("attn_fwd_c3_paged_b64.traffic.json", workload) == 1034019794
    said = bench.mfma_record(workload, 64, 1e9, 1.0, False)
    assert said["util"] == 0.1512 and "stale" not in said
