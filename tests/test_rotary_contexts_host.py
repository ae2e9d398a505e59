"""Contexts whose rotary positions have several axes ([axes, rows]): a decode context that follows such a prefill goes on from
its rotary positions, not from the tokens' places in the cache (state.decode_ctx_after, advance_decode_ctx)."""
import dataclasses

import pytest
import torch

from multi_modal_parallelism_b200.state import advance_decode_ctx, decode_ctx_after, make_prefill_ctx

CPU = torch.device("cpu")


def image_prefill(lens, starts=None, base=0):
    """Per sequence three text tokens, then rows of a grid four wide whose time stands still, all from `base` on."""
    pc = make_prefill_ctx(list(lens), 16, CPU, starts=starts, reserve=8)
    per = []
    for n in lens:
        t = torch.arange(n)
        grid = torch.stack([torch.full((n,), 3), 3 + (t - 3) // 4, 3 + (t - 3) % 4])
        per.append(torch.where(t < 3, t, grid) + base)
    return dataclasses.replace(pc, positions=torch.cat(per, 1)), per


@pytest.mark.parametrize("lens", [(12,), (5, 30, 3, 1)])
def test_decode_after_several_axes_goes_on_from_the_largest_position(lens):
    pc, per = image_prefill(lens)
    dc = decode_ctx_after(pc)
    want = torch.stack([p.max() + 1 for p in per]).expand(3, -1)
    assert dc.positions.dtype == torch.int64 and torch.equal(dc.positions, want)
    # where the token is cached and how many keys it sees follow its index, not its rotary position
    flat = decode_ctx_after(dataclasses.replace(pc, positions=make_prefill_ctx(list(lens), 16, CPU, reserve=8).positions))
    assert flat.positions.tolist() == list(lens)
    for name in ("slot_mapping", "seqused_k", "block_table", "state_idx", "cu_q"):
        assert torch.equal(getattr(dc, name), getattr(flat, name)), name
    assert (dc.c, dc.max_k, dc.B) == (flat.c, flat.max_k, flat.B)
    advance_decode_ctx(dc)
    advance_decode_ctx(flat)
    assert torch.equal(dc.positions, want + 1) and torch.equal(dc.slot_mapping, flat.slot_mapping)


def test_decode_after_a_continued_prefill_with_several_axes():
    pc, per = image_prefill((7, 12), starts=[20, 4], base=50)
    dc = decode_ctx_after(pc)
    assert torch.equal(dc.positions, torch.stack([p.max() + 1 for p in per]).expand(3, -1))
    assert dc.seqused_k.tolist() == [28, 17]


def test_sequences_without_new_tokens():
    """A fresh sequence without tokens starts at position 0; one that has cached tokens and no new ones gives no rotary
    position to go on from."""
    pc, per = image_prefill((7, 0))
    assert decode_ctx_after(pc).positions.tolist() == [[int(per[0].max()) + 1, 0]] * 3
    pc, _ = image_prefill((7, 0), starts=[0, 5])
    with pytest.raises(ValueError, match="rotary position"):
        decode_ctx_after(pc)


def test_positions_that_do_not_cover_the_rows_are_refused():
    pc, _ = image_prefill((7, 5))
    with pytest.raises(ValueError, match="positions"):
        decode_ctx_after(dataclasses.replace(pc, positions=pc.positions[:, :-1]))


def test_one_axis_layer_refuses_several_axes_on_every_prefill(monkeypatch):
    """Also where the buffers for that many rows are there already from a prefill with one axis."""
    from multi_modal_parallelism_b200 import layer as L
    from multi_modal_parallelism_b200.config import preset
    from multi_modal_parallelism_b200.dist import Coordinator, Groups
    from multi_modal_parallelism_b200.sharding import plan_for
    from multi_modal_parallelism_b200.state import alloc_states
    from multi_modal_parallelism_b200.weights import random_layer, shard_to_device
    from tests import _kernel_stand_ins as S

    monkeypatch.setattr(L, "K", S)
    dims = preset("hybrid_small")
    plan = plan_for("tp1", 0, 1, dims)
    pc = make_prefill_ctx([6, 3], 16, CPU)
    st = alloc_states(plan, dims, 3, pc.block_table.numel(), 16, CPU, torch.float32)
    groups = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=CPU)
    layer = L.ParallelHybridLayer(plan, shard_to_device(random_layer(dims, 0), plan, dims, CPU), dims, groups, st,
                                  decode_ctx_after(pc), CPU, overlap_branches=False)
    h = torch.randn(9, dims.hidden, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    several = dataclasses.replace(pc, positions=pc.positions.expand(3, -1))
    with pytest.raises(ValueError, match="one axis"):
        layer.prefill(h, several)
    first = layer.prefill(h, pc).clone()
    with pytest.raises(ValueError, match="one axis"):
        layer.prefill(h, several)
    assert torch.equal(layer.prefill(h, pc), first)


@pytest.mark.parametrize("sections", [(), (16, 8, 8)])
def test_a_refused_step_leaves_the_states_as_they_were(monkeypatch, sections):
    """Positions that the attention layer cannot take are found before the delta-rule layers ahead of it move their states."""
    from multi_modal_parallelism_b200 import qwen35 as Q
    from multi_modal_parallelism_b200.dist import Coordinator, Groups
    from tests import _kernel_stand_ins as S

    monkeypatch.setattr(Q, "K", S)
    d = Q.Qwen35Dims(hidden=256, n_k=4, n_v=8, n_q=4, n_kv=2, head_dim=64, intermediate=256, layout="GA", rope_sections=sections)
    g = Groups(rank=0, local_rank=0, world_size=1, tp=Coordinator((0,), None), pair=None, device=CPU)
    pc = make_prefill_ctx([9, 6], 16, CPU)
    stack = Q.Qwen35Stack(d, Q.random_stack(d, 0), "tp", g, CPU, 3, pc.block_table.numel(), 16, 40)
    x = torch.randn(15, d.hidden, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    for ctx, n in ((pc, 15), (decode_ctx_after(pc), 2)):
        for shape in [(n - 1,), (2 * n,), (3, n - 1), (2, n), (3, 2, n)] + ([] if sections else [(3, n)]):
            with pytest.raises(ValueError, match="positions"):
                stack.step(x[:n], dataclasses.replace(ctx, positions=torch.ones(shape, dtype=torch.int64)))
    gdn = stack.layers[0]
    assert not bool(gdn.ssm_state.any()) and not bool(gdn.conv_state.any())
    stack.step(x, pc)
    assert bool(gdn.ssm_state.any())
