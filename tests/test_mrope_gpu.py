"""Rotary positions with several axes and the paged cache write (kernels.qkv_mrope_kv_write) on one B200 against the formula
in 64 bits. Tolerance: the rounding to bf16 (2^-8 of the value) plus, for a value a c - b s, the fp32 errors of c and s (the
reduced angle's rounding, 2^-23 of at most pi, and sincosf's 2 units) and of the two products: (|a| + |b|) 2^-20. Passed
dims and values are exact where no multiplier applies."""
import pytest
import torch

from multi_modal_parallelism_b200 import kernels as K
from multi_modal_parallelism_b200._lib import MmpError
from multi_modal_parallelism_b200.state import alloc_kv

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    torch.cuda.synchronize()
    K.check_device_errors(DEV)


def case(T, nq, nkv, hd, rd, A, interleaved, block, seed=0, start=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    half = rd // 2
    sec = [half - (A - 1) * (half // 4)] + [half // 4] * (A - 1) if half >= 4 else [half] + [0] * (A - 1)
    c = {"qkv": torch.randn(T, (nq + 2 * nkv) * hd, generator=g).to(BF).to(DEV),
         "positions": (torch.randint(0, 1000, (A, T), generator=g) + start).to(DEV),
         "inv_freq": K.rope_inv_freq(rd, 1e4, DEV), "axes": K.rope_axes(sec, interleaved, DEV)}
    nb = -(-T // block) + 1
    c["kv"], c["key_cache"], c["value_cache"], _ = alloc_kv(nb, block, nkv, hd, DEV)
    slots = torch.randperm(nb * block, generator=g)[:T]
    if pad:
        slots[-pad:] = -1
    c["slots"] = slots.to(DEV)
    c["q_out"] = torch.full((T, nq * hd), 5.0, dtype=BF, device=DEV)
    return c


def run(c, nq, nkv, hd, mult=0.75):
    return K.qkv_mrope_kv_write(c["qkv"], nq, nkv, hd, c["positions"], c["inv_freq"], c["axes"], mult, c["q_out"], c["key_cache"],
                                c["value_cache"], c["slots"])


def check(c, qkv, nq, nkv, hd, mult=0.75):
    half, T = c["inv_freq"].numel(), qkv.shape[0]
    x = qkv.double().view(T, nq + 2 * nkv, hd)
    ang = c["positions"][c["axes"].long()].T.double() * c["inv_freq"].double()
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    m = torch.ones(nq + nkv, 1, dtype=torch.float64, device=DEV)
    m[nq:] = float(torch.tensor(mult))
    qk = x[:, :nq + nkv] * m
    a, b = qk[..., :half], qk[..., half:2 * half]
    ref = torch.cat([a * cos - b * sin, b * cos + a * sin, qk[..., 2 * half:]], -1)
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    tol = 2.0 ** -8 * ref.abs()
    tol[..., :2 * half] += 2.0 ** -20 * size
    q = c["q_out"].double().view(T, nq, hd)
    assert bool(((q - ref[:, :nq]).abs() <= tol[:, :nq]).all())
    ok = c["slots"] >= 0
    s, block = c["slots"][ok], c["key_cache"].shape[1]
    k = c["key_cache"][s // block, s % block].double()
    assert bool(((k - ref[:, nq:][ok]).abs() <= tol[:, nq:][ok]).all())
    assert torch.equal(c["value_cache"][s // block, s % block], qkv.view(T, nq + 2 * nkv, hd)[:, nq + nkv:][ok])
    untouched = torch.ones(c["kv"].shape[0] * block, dtype=torch.bool, device=DEV)
    untouched[s] = False
    assert not bool(c["kv"].transpose(1, 2).reshape(-1, nkv, 2 * hd)[untouched].any())


@pytest.mark.parametrize("T,nq,nkv,hd,rd,A,interleaved,block", [
    (1, 1, 1, 64, 64, 1, False, 16), (1, 16, 2, 128, 128, 3, True, 16), (7, 4, 2, 128, 64, 3, False, 16), (65, 16, 2, 256, 64, 3, True, 64),
    (130, 8, 8, 64, 16, 2, True, 32), (33, 3, 1, 80, 80, 3, False, 16), (20, 2, 1, 72, 36, 2, False, 16), (9, 2, 1, 20, 6, 1, False, 16),
    (300, 32, 8, 128, 128, 3, True, 16), (5, 6, 2, 128, 2, 1, True, 1)])
def test_matches_formula(T, nq, nkv, hd, rd, A, interleaved, block):
    c = case(T, nq, nkv, hd, rd, A, interleaved, block, seed=T)
    assert run(c, nq, nkv, hd) is c["q_out"]
    check(c, c["qkv"], nq, nkv, hd)


@pytest.mark.parametrize("start", [10 ** 6, 2 ** 31 + 5, 10 ** 10])
def test_far_positions_keep_their_angle(start):
    c = case(40, 4, 2, 128, 128, 3, True, 16, start=start)
    run(c, 4, 2, 128)
    check(c, c["qkv"], 4, 2, 128)


def test_padding_rows_are_rotated_and_not_cached():
    c = case(40, 4, 2, 128, 64, 3, True, 16, pad=9)
    run(c, 4, 2, 128)
    check(c, c["qkv"], 4, 2, 128)


def test_equal_axes_match_the_single_axis_kernel():
    """The same position on every axis is the one-axis rotation (whose fp32 angle agrees to 2^-15 below position 1000)."""
    c = case(50, 4, 2, 128, 128, 3, True, 16)
    c["positions"] = c["positions"][:1].expand(3, -1).contiguous()
    run(c, 4, 2, 128)
    kv, kc, vc, _ = alloc_kv(c["kv"].shape[0], 16, 2, 128, DEV)
    q = torch.empty_like(c["q_out"])
    K.qkv_rope_kv_write(c["qkv"], 4, 2, 128, c["positions"][0].contiguous(), c["inv_freq"], 0.75, q, kc, vc, c["slots"])
    for a, b in ((q, c["q_out"]), (kv, c["kv"])):
        assert bool(((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -10).all())


@pytest.mark.parametrize("shift", [0, 1])
def test_strided_rows_in_place_queries_and_odd_offsets(shift):
    """q written over the projection's own q columns; shift 1 starts the rows off a 16-byte boundary."""
    T, nq, nkv, hd = 21, 4, 2, 64
    c = case(T, nq, nkv, hd, 64, 3, True, 16)
    buf = torch.full((T, (nq + 2 * nkv) * hd + 16), 7.0, dtype=BF, device=DEV)
    qkv = buf[:, shift:shift + (nq + 2 * nkv) * hd].copy_(c["qkv"])
    before = c["qkv"]
    c["qkv"], c["q_out"] = qkv, qkv[:, :nq * hd]
    run(c, nq, nkv, hd)
    check({**c, "q_out": c["q_out"].contiguous()}, before, nq, nkv, hd)
    assert torch.equal(qkv[:, nq * hd:], before[:, nq * hd:]) and bool((buf[:, shift + qkv.shape[1]:] == 7).all())


def test_cache_of_another_layout():
    """Key and value caches as plain [blocks, block, heads, dim] tensors."""
    T, nq, nkv, hd = 30, 4, 2, 128
    c = case(T, nq, nkv, hd, 128, 3, False, 16)
    c["key_cache"], c["value_cache"] = (torch.zeros(3, 16, nkv, hd, dtype=BF, device=DEV) for _ in range(2))
    run(c, nq, nkv, hd)
    c["kv"] = torch.cat([c["key_cache"], c["value_cache"]], -1).transpose(1, 2)
    check(c, c["qkv"], nq, nkv, hd)


def test_slot_past_the_cache_and_bad_axis_are_reported():
    c = case(10, 2, 1, 64, 64, 2, True, 16)
    good = c["slots"].clone()
    c["slots"][3] = c["kv"].shape[0] * 16
    run(c, 2, 1, 64)
    with pytest.raises(MmpError, match="index out of range"):
        K.check_device_errors(DEV)
    c["slots"] = good
    c["slots"][3] = -1
    check(c, c["qkv"], 2, 1, 64)
    c = case(10, 2, 1, 64, 64, 2, True, 16)
    c["axes"][0] = 2
    run(c, 2, 1, 64)
    with pytest.raises(MmpError, match="index out of range"):
        K.check_device_errors(DEV)


def test_captured_and_replayed():
    c = case(12, 4, 2, 128, 128, 3, True, 16)
    run(c, 4, 2, 128)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(c, 4, 2, 128)
    c["qkv"].copy_(torch.randn(c["qkv"].shape, generator=torch.Generator().manual_seed(9)))
    c["positions"].add_(17)
    graph.replay()
    torch.cuda.synchronize()
    check(c, c["qkv"], 4, 2, 128)


def test_empty_batch():
    c = case(1, 2, 1, 64, 64, 1, False, 16)
    K.qkv_mrope_kv_write(c["qkv"][:0], 2, 1, 64, c["positions"][:, :0], c["inv_freq"], c["axes"], 1.0, c["q_out"][:0], c["key_cache"],
                         c["value_cache"], c["slots"][:0])
