"""bench.py's rate of a kernel that is bound by the MXFP4 tensor cores."""
import importlib.util
from pathlib import Path

import pytest


def test_benchmark_rows_of_mxfp4_kernels_have_a_rate():
    spec = importlib.util.spec_from_file_location("bench_module", Path(__file__).resolve().parents[1] / "bench.py")
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    pk = {"hbm_gbs": 6000.0, "bf16_burst": 1700.0, "bf16_sustained": 1400.0, "source": "measured"}
    row = bench.kernel_row("g", "b2_mxfp4_gemm", 1.0, "mxfp4", 3_400_000_000_000, pk)
    assert row["achieved"] == pytest.approx(3400.0) and row["frac"] == pytest.approx(0.5) and "ASSUMED" in row["peak_kind"]
