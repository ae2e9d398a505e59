import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


# Tests whose calls pass the library's argument checks with CPU tensors and count on the launch to fail: with a GPU the kernels
# would read host addresses (an illegal access).
HOST_ONLY = ("test_abi_validation.py::", "test_ssd_segments_host.py::test_segmented_prefill_calls_validate")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (CUDA sm_100a) and the built libmmp_b200.so")
    config.addinivalue_line("markers", "run_last(order=0): collected after every other test, so that under -x a "
                                       "failure there cannot hide the results of the rest of the suite; among "
                                       "them, higher orders run later")


def _run_last_key(it) -> tuple[int, int]:
    m = it.get_closest_marker("run_last")
    if m is None:
        return (0, 0)
    return (1, int(m.kwargs.get("order", m.args[0] if m.args else 0)))


def pytest_collection_modifyitems(config, items):
    items.sort(key=_run_last_key)  # stable: file order otherwise kept
    # GPU tests are skipped, not failed, where no GPU is visible (the CPU suite runs everything else).
    try:
        import torch

        has_gpu = torch.cuda.is_available()
    except Exception:  # pragma: no cover
        has_gpu = False
    if has_gpu:
        skip = pytest.mark.skip(reason="hands CPU tensors to the library: runs on a machine without a GPU")
        for it in items:
            if f"{it.path.name}::{it.name}".startswith(HOST_ONLY):
                it.add_marker(skip)
        return
    skip = pytest.mark.skip(reason="no CUDA device visible")
    for it in items:
        if "gpu" in it.keywords:
            it.add_marker(skip)


def _stood_in():
    """The package's modules whose `K` is not the kernels module."""
    K = sys.modules.get("multi_modal_parallelism_b200.kernels")
    return [m for n, m in list(sys.modules.items()) if n.startswith("multi_modal_parallelism_b200.") and K is not None
            and getattr(m, "K", K) is not K]


@pytest.fixture(autouse=True)
def _kernels_module(request):
    """Host tests may assign stand-ins for the kernels module (`qwen35.K = ...`): they end with the test, and no GPU test starts
    with one."""
    if request.node.get_closest_marker("gpu"):
        assert not _stood_in(), [m.__name__ for m in _stood_in()]
    yield
    for m in _stood_in():
        m.K = sys.modules["multi_modal_parallelism_b200.kernels"]
