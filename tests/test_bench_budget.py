"""How long `python bench.py` takes: its long extras are sized against a budget that ends before ten minutes do, so that the line is printed."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def test_the_default_budget_leaves_no_room_for_what_takes_longer():
    import bench

    budget = bench.arguments().parse_args([]).budget_s
    assert budget <= 560
    # a graph of 10 M x 768 rows takes 350 s and its ground truth, records and searches 60 more; the points before it take 300 s
    assert bench.config4_vectors(10_000_000, budget - 300, 280e9)[0] == 2_000_000
    assert bench.config4_vectors(10_000_000, 1500 - 300, 280e9) == (10_000_000, None)
    assert bench.config4_vectors(10_000_000, 1500, 100e9)[0] == 2_000_000 and "GB" in bench.config4_vectors(10_000_000, 1500, 100e9)[1]
    assert bench.config4_vectors(2_000_000, 10, 1e9) == (2_000_000, None)


def test_the_budget_can_be_given():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--help"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "--budget-s" in out.stdout + out.stderr
