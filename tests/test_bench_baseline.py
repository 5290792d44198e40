"""CPU: the benchmark says why a run has no CPU figure of the reference."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_missing_baseline_is_named(monkeypatch):
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    import bench
    res = {}
    monkeypatch.setattr(bench, "ref_missing", lambda: "not built")
    bench.add_cpu_baseline(res, lambda: 1 / 0)  # not measured
    assert res == {"cpu_baseline_unavailable": "not built"}
    res = {}
    monkeypatch.setattr(bench, "ref_missing", lambda: None)
    bench.add_cpu_baseline(res, lambda: {"value": 3})
    assert res == {"cpu_baseline": {"value": 3}}
