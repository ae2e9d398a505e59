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


@pytest.mark.parametrize("rotary", [-2, 1, 63, 65, 130, 128])
def test_rotation_of_more_dims_than_a_head_or_of_an_odd_number_is_refused(monkeypatch, rotary):
    from multi_modal_parallelism_b200 import qwen35 as Q
    from multi_modal_parallelism_b200.dist import Coordinator, Groups
    from tests import _kernel_stand_ins as S

    monkeypatch.setattr(Q, "K", S)
    dev = torch.device("cpu")
    g = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=dev)
    d = Q.Qwen35Dims(hidden=256, n_q=4, n_kv=2, head_dim=64, intermediate=64, layout="A")
    for ok in (0, 2, 32, 64):
        Q.Qwen35Stack(d.replace(rotary_dim=ok), Q.random_stack(d, 0), "tp", g, dev, 2, 4, 16, 8)
    with pytest.raises(ValueError, match="rotary_dim"):
        Q.Qwen35Stack(d.replace(rotary_dim=rotary), Q.random_stack(d, 0), "tp", g, dev, 2, 4, 16, 8)


def test_a_step_of_more_rows_than_the_stack_has_is_refused(monkeypatch):
    from multi_modal_parallelism_b200 import qwen35 as Q
    from multi_modal_parallelism_b200.dist import Coordinator, Groups
    from multi_modal_parallelism_b200.state import make_prefill_ctx
    from tests import _kernel_stand_ins as S

    monkeypatch.setattr(Q, "K", S)
    dev = torch.device("cpu")
    g = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=dev)
    d = Q.Qwen35Dims(hidden=256, n_k=4, n_v=8, n_q=4, n_kv=2, head_dim=64, layout="GA", n_experts=4, top_k=2, moe_intermediate=64)
    stack = Q.Qwen35Stack(d, Q.random_stack(d, 0), "tp", g, dev, 2, 4, 16, 8)
    x = torch.zeros(9, d.hidden, dtype=BF)
    stack.step(x[:8], make_prefill_ctx([8], 16, dev))
    with pytest.raises(ValueError, match="max_tokens"):
        stack.step(x, make_prefill_ctx([9], 16, dev))
