"""Tests that hand CPU tensors to the library and rely on its launches failing (no GPU) do not run where a GPU is visible: their
kernels would read host addresses there."""
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
RUN = ("import sys, torch, pytest; torch.cuda.is_available = lambda: True; "
       "sys.exit(pytest.main(['-q', '-rs', '-p', 'no:cacheprovider', *sys.argv[1:]]))")


@pytest.mark.parametrize("tests,n", [
    ("tests/test_abi_validation.py::test_hybrid_layer_calls_validate", 3),
    ("tests/test_abi_validation.py::test_a_misaligned_request_is_caught", 1),
    ("tests/test_ssd_segments_host.py::test_segmented_prefill_calls_validate", 1),
])
def test_skipped_where_a_gpu_is_visible(tests, n):
    r = subprocess.run([sys.executable, "-c", RUN, tests], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and f"{n} skipped" in r.stdout and "without a GPU" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_others_run_there():
    r = subprocess.run([sys.executable, "-c", RUN, "tests/test_ssd_segments_host.py::test_build_segments_arrays"], cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "1 passed" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
