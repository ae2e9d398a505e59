"""Calls of the mixture-of-experts wrappers and of the stack around them that have to be refused before a launch, on a machine
without a GPU (the wrappers run with CPU tensors and only their device assertion relaxed)."""
import pytest
import torch

from multi_modal_parallelism_b200 import kernels as K
from tests.test_moe_host import BF, E, H, I, T, cpu, experts, k  # noqa: F401 (cpu: a fixture)

ROOM = 1 << 20


def aligned(n):
    t = torch.zeros(n + 256, dtype=torch.uint8)
    return t[-t.data_ptr() % 256:][:n]


@pytest.mark.parametrize("scratch", [
    aligned(256).expand(ROOM // 256, 256),       # more elements than bytes behind them
    aligned(1).expand(ROOM),
    aligned(2 * ROOM)[::2],
    aligned(2 * ROOM).view(1024, 2048)[:, :1024],
], ids=["rows", "one", "every-second", "columns"])
def test_scratch_with_gaps_or_repeats_is_refused(cpu, scratch):  # noqa: F811
    a = experts()
    with pytest.raises(ValueError, match="workspace"):
        K.moe_experts(**experts(workspace=scratch))
    with pytest.raises(ValueError, match="workspace"):
        K.moe_layer(a["x"], torch.zeros(T, E), a["w_gate_up"], a["w_down"], k, workspace=scratch)
