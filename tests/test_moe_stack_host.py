"""Host logic of the stack with a mixture of experts and several-axis rotary positions (multi_modal_parallelism_b200.qwen35)
on CPU ranks: every expert's columns split over the ranks, the router replicated, the shared expert behind the routed ones,
rotary positions kept apart from cache slots. The kernel wrappers are torch stand-ins; a prefill of two ragged sequences
with image-like positions, then decode steps, against the numpy stack oracle: max-abs <= 2e-2 * max(1, max|ref|), rel-L2
<= 1e-2. Every expert is chosen (top_k = experts), so that no rounding turns a choice."""
import dataclasses
import multiprocessing as mp
import os
import socket

import numpy as np
import pytest
import torch

import oracle
from multi_modal_parallelism_b200.correctness import compare, within_tolerance
from multi_modal_parallelism_b200.qwen35 import Qwen35Dims, mlp_cols, random_stack

DIMS = Qwen35Dims(hidden=256, n_k=4, n_v=8, n_q=4, n_kv=2, layout="GA", n_experts=4, top_k=4, moe_intermediate=64,
                  shared_expert=True, rotary_dim=64, rope_sections=(16, 8, 8))
LENS, STEPS, SEED, KV_BLOCK = (9, 6), 2, 3, 16


def weights():
    ws = random_stack(DIMS, SEED)
    for w in ws:
        for k in list(w):
            if k in ("self_attn.q_proj.weight", "self_attn.k_proj.weight", "mlp.gate.weight", "mlp.shared_expert_gate.weight"):
                w[k] = (w[k].float() * 12).to(torch.bfloat16)  # scores and router logits of order one
            if k.startswith("mlp.experts") or k.startswith("mlp.shared_expert."):
                w[k] = (w[k].float() * 4).to(torch.bfloat16)
    return ws


def positions():
    """Prefill [axes, T] and per step [axes, sequences]: a few text tokens, then a 2 x 2 grid whose time stands still, so
    that the rotary positions fall behind the token indices."""
    per = []
    for L in LENS:
        t = np.arange(L)
        g = np.stack([np.full(L, 3), 3 + (t - 3) // 2 % 2, 3 + (t - 3) % 2])
        per.append(np.where(t < 3, t, g))
    steps = [np.tile([6 + s, 5 + s], (3, 1)) for s in range(STEPS)]
    return per, steps


def inputs():
    g = torch.Generator().manual_seed(SEED + 7)
    hp = torch.randn(sum(LENS), DIMS.hidden, generator=g).to(torch.bfloat16)
    return hp, [torch.randn(len(LENS), DIMS.hidden, generator=g).to(torch.bfloat16) for _ in range(STEPS)]


def run_rank(mode, groups):
    from multi_modal_parallelism_b200 import qwen35 as Q
    from multi_modal_parallelism_b200.state import advance_decode_ctx, decode_ctx_after, make_prefill_ctx
    from tests import _kernel_stand_ins as S

    Q.K = S  # torch stand-ins for the CUDA kernels (test only)
    cpu = torch.device("cpu")
    per, steps = positions()
    pc = make_prefill_ctx(list(LENS), KV_BLOCK, cpu, reserve=STEPS + 1)
    pc = dataclasses.replace(pc, positions=torch.from_numpy(np.concatenate(per, 1)))
    stack = Q.Qwen35Stack(DIMS, weights(), mode, groups, cpu, lines=len(LENS) + 1, num_blocks=pc.block_table.numel(),
                          kv_block=KV_BLOCK, max_tokens=sum(LENS))
    hp, hd = inputs()
    outs = [stack.step(hp, pc).float().numpy().copy()]
    dc = dataclasses.replace(decode_ctx_after(pc), positions=torch.from_numpy(steps[0]))
    for s in range(STEPS):
        assert np.array_equal(dc.positions.numpy(), steps[s])
        outs.append(stack.step(hd[s], dc).float().numpy().copy())
        advance_decode_ctx(dc)
    return outs


def reference_outputs():
    ws = [{k: oracle.to_numpy(v) for k, v in w.items()} for w in weights()]
    hp, hd = inputs()
    hp = hp.float().numpy()
    cu = np.concatenate([[0], np.cumsum(LENS)])
    per, steps = positions()
    outs, state = oracle.qwen35_stack_prefill(ws, DIMS, [hp[cu[i]:cu[i + 1]] for i in range(len(LENS))], positions=per)
    refs = [np.concatenate(outs, 0)]
    for s in range(STEPS):
        o, state = oracle.qwen35_stack_decode(ws, DIMS, hd[s].float().numpy(), state, positions=steps[s])
        refs.append(o)
    return refs


def check(outs, refs, what):
    for i, (o, r) in enumerate(zip(outs, refs)):
        m = compare(torch.from_numpy(o), torch.from_numpy(r))
        assert within_tolerance(m), f"{what} call {i}: {m}"


def test_single_rank():
    from multi_modal_parallelism_b200.dist import Coordinator, Groups

    g = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=torch.device("cpu"))
    check(run_rank("tp", g), reference_outputs(), "world 1")


def test_expert_columns_split_in_multiples_of_eight():
    assert [list(mlp_cols(DIMS, r, 2)) for r in range(2)] == [list(range(32)), list(range(32, 64))]
    with pytest.raises(ValueError):
        mlp_cols(DIMS.replace(moe_intermediate=24), 0, 2)


def test_rotary_sections_that_do_not_fill_the_rotation_are_refused():
    from multi_modal_parallelism_b200 import qwen35 as Q
    from multi_modal_parallelism_b200.dist import Coordinator, Groups
    from tests import _kernel_stand_ins as S

    Q.K = S
    g = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=torch.device("cpu"))
    d = DIMS.replace(rope_sections=(16, 8, 4), layout="A")
    with pytest.raises(ValueError, match="rope_sections"):
        Q.Qwen35Stack(d, random_stack(d, 0), "tp", g, torch.device("cpu"), 2, 4, 16, 8)


def test_positions_with_several_axes_are_refused_where_the_rotation_has_one():
    from types import SimpleNamespace

    from multi_modal_parallelism_b200 import qwen35 as Q
    from multi_modal_parallelism_b200.dist import Coordinator, Groups
    from multi_modal_parallelism_b200.layer import AttentionBranch
    from multi_modal_parallelism_b200.state import make_prefill_ctx
    from tests import _kernel_stand_ins as S

    Q.K = S
    cpu = torch.device("cpu")
    g = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=cpu)
    d = DIMS.replace(rope_sections=(), rotary_dim=0, layout="A")
    ctx = make_prefill_ctx([8], 16, cpu)
    several = dataclasses.replace(ctx, positions=ctx.positions.expand(3, -1))
    stack = Q.Qwen35Stack(d, random_stack(d, 0), "tp", g, cpu, 2, 4, 16, 8)
    x = torch.zeros(8, d.hidden, dtype=torch.bfloat16)
    stack.step(x, ctx)
    with pytest.raises(ValueError, match="one axis"):
        stack.step(x, several)
    plan = SimpleNamespace(attn=SimpleNamespace(q_heads=[0], kv_heads=[0]))
    with pytest.raises(ValueError, match="one axis"):
        AttentionBranch(plan, None, None, None, several, cpu)


def test_yaml_of_the_moe_stack():
    d = Qwen35Dims.from_yaml("qwen35_moe_like")
    assert (d.n_experts, d.top_k, d.moe_intermediate, d.shared_expert) == (256, 8, 512, True)
    assert d.rope_sections == (24, 20, 20) and sum(d.rope_sections) == d.head_dim // 2
    assert Qwen35Dims.from_yaml("qwen35_like").n_experts == 0


def _free_port() -> int:
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _worker(rank, world, port, mode, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank))
    torch.set_num_threads(1)
    try:
        from multi_modal_parallelism_b200.dist import destroy, init_groups

        groups = init_groups(backend="gloo", timeout_s=120)
        q.put((rank, run_rank(mode, groups), None))
        destroy()
    except Exception as e:  # pragma: no cover - reported to the parent
        import traceback

        q.put((rank, None, traceback.format_exc()[-2000:] + repr(e)))


@pytest.mark.parametrize("mode", ["tp", "attn_dp"])
def test_two_ranks(mode):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, mode, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted((q.get(timeout=300) for _ in range(2)), key=lambda r: r[0])
    for p in procs:
        p.join(timeout=60)
    for rank, _, err in res:
        assert err is None, f"rank {rank}: {err}"
    refs = reference_outputs()
    for rank, outs, _ in res:
        check(outs, refs, f"{mode} rank {rank}")
        assert all(np.array_equal(o, o0) for o, o0 in zip(outs, res[0][1]))
