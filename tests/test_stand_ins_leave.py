"""Host tests put torch stand-ins in the place of the kernels module (`qwen35.K = ...`). None of them outlives its test: a GPU test
that runs later in the same process would pass without launching a kernel."""
import subprocess
import sys
from pathlib import Path

import pytest

from multi_modal_parallelism_b200 import kernels, layer, mamba2, qwen35

ROOT = Path(__file__).resolve().parents[1]


def test_modules_use_the_kernels():
    """Run by itself, and by the tests below after tests that use stand-ins."""
    for m in (qwen35, layer, mamba2):
        assert m.K is kernels, f"{m.__name__} still uses {m.K.__name__}"


@pytest.mark.parametrize("before", [
    "test_moe_stack_host.py::test_single_rank",
    "test_moe_stack_host.py::test_rotary_sections_that_do_not_fill_the_rotation_are_refused",
    "test_moe_stack_host.py::test_positions_with_several_axes_are_refused_where_the_rotation_has_one",
    "test_qwen35_host.py::test_single_rank",
    "test_mamba2_layer_host.py::test_single_rank_tp",
])
def test_stand_ins_do_not_outlive_their_test(before):
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", f"tests/{before}",
                        "tests/test_stand_ins_leave.py::test_modules_use_the_kernels"], cwd=ROOT, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0 and "2 passed" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
