"""The stack with a mixture of experts and several-axis rotary positions on one B200: the operators run together as a model
uses them. (1) A prefill of three ragged sequences with image-like positions, then decode steps, against the numpy stack
oracle, every expert chosen (top_k = experts) so that no rounding turns a choice; (2) with fewer experts chosen, each MoE
layer against the formula on the layer's own inputs and logits. Tolerance: max-abs <= 2e-2 * max(1, max|ref|), rel-L2 <=
1e-2. (3) A decode step captured into a CUDA graph gives the eager step's bits."""
import dataclasses

import numpy as np
import pytest
import torch

import oracle
from multi_modal_parallelism_b200 import kernels as K
from multi_modal_parallelism_b200.correctness import compare, describe, within_tolerance
from multi_modal_parallelism_b200.dist import Coordinator, Groups
from multi_modal_parallelism_b200.qwen35 import Qwen35Dims, Qwen35Stack, random_stack
from multi_modal_parallelism_b200.state import advance_decode_ctx, decode_ctx_after, make_prefill_ctx
from oracle.moe import moe_mlp

pytestmark = [pytest.mark.gpu, pytest.mark.run_last]
DEV = torch.device("cuda", 0)
DIMS = Qwen35Dims(hidden=512, n_k=2, n_v=4, n_q=4, n_kv=2, layout="GA", n_experts=4, top_k=4, moe_intermediate=128,
                  shared_expert=True, rotary_dim=64, rope_sections=(16, 8, 8))
LENS, STEPS, SEED, KV_BLOCK = (100, 37, 64), 3, 5, 16


def weights(d):
    ws = random_stack(d, SEED)
    for w in ws:
        for k in list(w):
            if k in ("self_attn.q_proj.weight", "self_attn.k_proj.weight", "mlp.gate.weight", "mlp.shared_expert_gate.weight"):
                w[k] = (w[k].float() * 2.2).to(torch.bfloat16)  # scores and router logits of order one
            if k.startswith("mlp.experts") or k.startswith("mlp.shared_expert."):
                w[k] = (w[k].float() * 2.5).to(torch.bfloat16)
    return ws


def positions(lens, steps):
    per = []
    for L in lens:
        t = np.arange(L)
        g = np.stack([np.full(L, 5), 5 + (t - 5) // 8, 5 + (t - 5) % 8])
        per.append(np.where(t < 5, t, g))
    last = [p.max() + 1 for p in per]
    return per, [np.tile(np.array(last) + s, (3, 1)) for s in range(steps)]


def build(d, ws, lens, reserve=STEPS + 1):
    groups = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=DEV)
    pc = make_prefill_ctx(list(lens), KV_BLOCK, DEV, reserve=reserve)
    per, steps = positions(lens, STEPS)
    pc = dataclasses.replace(pc, positions=torch.from_numpy(np.concatenate(per, 1)).to(DEV))
    stack = Qwen35Stack(d, ws, "tp", groups, DEV, lines=len(lens) + 1, num_blocks=pc.block_table.numel(), kv_block=KV_BLOCK,
                        max_tokens=sum(lens))
    dc = dataclasses.replace(decode_ctx_after(pc), positions=torch.from_numpy(steps[0]).to(DEV))
    return stack, pc, dc, per, steps


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    K.check_device_errors(DEV)


def test_prefill_then_decode_matches_oracle():
    g = torch.Generator().manual_seed(SEED + 7)
    hp = torch.randn(sum(LENS), DIMS.hidden, generator=g).to(torch.bfloat16)
    hd = [torch.randn(len(LENS), DIMS.hidden, generator=g).to(torch.bfloat16) for _ in range(STEPS)]
    ws = weights(DIMS)
    stack, pc, dc, per, steps = build(DIMS, ws, LENS)
    outs = [stack.step(hp.to(DEV), pc).float().cpu().numpy()]
    for s in range(STEPS):
        outs.append(stack.step(hd[s].to(DEV), dc).float().cpu().numpy())
        advance_decode_ctx(dc)
    wn = [{k: oracle.to_numpy(v) for k, v in w.items()} for w in ws]
    cu = np.concatenate([[0], np.cumsum(LENS)])
    hpn = hp.float().numpy()
    ref, state = oracle.qwen35_stack_prefill(wn, DIMS, [hpn[cu[i]:cu[i + 1]] for i in range(len(LENS))], positions=per)
    refs = [np.concatenate(ref, 0)]
    for s in range(STEPS):
        o, state = oracle.qwen35_stack_decode(wn, DIMS, hd[s].float().numpy(), state, positions=steps[s])
        refs.append(o)
    for i, (o, r) in enumerate(zip(outs, refs)):
        m = compare(torch.from_numpy(o), torch.from_numpy(r))
        assert within_tolerance(m), f"call {i}: {describe(m)}"


@pytest.mark.parametrize("lens", [LENS, (400, 300, 500)])
def test_each_layers_experts_on_its_own_logits(lens):
    d = DIMS.replace(n_experts=24, top_k=4)
    ws = weights(d)
    stack, pc, dc, _, _ = build(d, ws, lens)
    g = torch.Generator().manual_seed(SEED)
    h = torch.randn(sum(lens), d.hidden, generator=g).to(torch.bfloat16).to(DEV)
    for ctx, x in ((pc, h), (dc, h[:len(lens)])):
        for layer, w in zip(stack.layers, ws):
            x = layer.step(x, ctx)
            T = x.shape[0]
            wn = {k: oracle.to_numpy(v) for k, v in w.items()}
            logits = layer.mlp.logits[:T, :25].float().cpu().numpy()
            ref = layer.h1[:T].float().cpu().numpy() + moe_mlp(wn, d, layer.y[:T].float().cpu().numpy(), logits)
            m = compare(x.float().cpu(), torch.from_numpy(ref))
            assert within_tolerance(m), describe(m)


def test_decode_step_captured_into_a_graph():
    d = DIMS.replace(n_experts=24, top_k=4)
    stack, pc, dc, _, _ = build(d, weights(d), LENS)
    g = torch.Generator().manual_seed(SEED)
    stack.step(torch.randn(sum(LENS), d.hidden, generator=g).to(torch.bfloat16).to(DEV), pc)
    x = torch.randn(len(LENS), d.hidden, generator=g).to(torch.bfloat16).to(DEV)
    states = [(t, t.clone()) for layer in stack.layers for t in (getattr(layer, "ssm_state", None), getattr(layer, "conv_state", None))
              if t is not None]
    eager = stack.step(x, dc).clone()
    for t, t0 in states:
        t.copy_(t0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = stack.step(x, dc)
    for t, t0 in states:
        t.copy_(t0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
