"""The mixture-of-experts layers of a stack run one after another and share one scratch (at 16384 rows of 9 places, hidden 2048,
intermediate 512 it is 2 GB). CPU, torch stand-ins for the kernel wrappers."""
import pytest
import torch

from multi_modal_parallelism_b200 import _lib
from multi_modal_parallelism_b200 import qwen35 as Q
from multi_modal_parallelism_b200.dist import Coordinator, Groups
from multi_modal_parallelism_b200.state import decode_ctx_after, make_prefill_ctx
from tests import _kernel_stand_ins as S

CPU = torch.device("cpu")
DIMS = Q.Qwen35Dims(hidden=256, n_k=4, n_v=8, n_q=4, n_kv=2, layout="GAG", n_experts=4, top_k=2, moe_intermediate=64)


@pytest.mark.parametrize("shared", [False, True])
def test_one_scratch_for_all_layers(monkeypatch, shared):
    sized, used = [], []

    def workspace(*size):
        sized.append(size[:5])
        return torch.empty(1)

    def layer(*a, workspace=None, **kw):
        used.append(workspace)
        return moe_layer(*a, workspace=workspace, **kw)

    moe_layer = S.moe_layer
    monkeypatch.setattr(S, "moe_workspace", workspace)
    monkeypatch.setattr(S, "moe_layer", layer)
    monkeypatch.setattr(Q, "K", S)
    d = DIMS.replace(shared_expert=shared)
    groups = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=CPU)
    pc = make_prefill_ctx([9, 6], 16, CPU)
    stack = Q.Qwen35Stack(d, Q.random_stack(d, 0), "tp", groups, CPU, 3, pc.block_table.numel(), 16, 40)
    x = torch.randn(15, d.hidden).to(torch.bfloat16)
    stack.step(x, pc)
    stack.step(x[:2], decode_ctx_after(pc))
    # of the largest call: max_tokens rows, the chosen experts' places and the shared one's
    assert sized == [(40, 2 + shared, 256, 64, 4 + shared)]
    assert len(used) == 6 and all(u is used[0] for u in used)


def test_a_dense_stack_has_none(monkeypatch):
    monkeypatch.setattr(S, "moe_workspace", lambda *a: pytest.fail("scratch without experts"))
    monkeypatch.setattr(Q, "K", S)
    d = DIMS.replace(n_experts=0, intermediate=256)
    groups = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=CPU)
    Q.Qwen35Stack(d, Q.random_stack(d, 0), "tp", groups, CPU, 3, 4, 16, 40)


def test_scratch_of_a_long_prompt_is_gigabytes():
    """What a second one would cost: fp32 results and bf16 rows of 16384 x 9 places."""
    n = _lib.lib().mmp_moe_workspace_size(16384, 9, 2048, 512, 257)
    assert n >= 16384 * 9 * (2048 * 4 + 2048 * 2 + 512 * 2)
