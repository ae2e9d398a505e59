"""Far positions of kernels.qkv_mrope_kv_write on one B200. The reference angle is taken in integers: position times the fp32
frequency exactly, modulo 2 pi to 200 bits. Tolerance as for near positions: the rounding to bf16 (2^-8 of the value) and, for
a value a c - b s, (|a| + |b|) 2^-20 for the fp32 angle, its sine and cosine and the two products."""
import math

import pytest
import torch

from tests.test_mrope_gpu import DEV, case, run

from multi_modal_parallelism_b200 import kernels as K

pytestmark = pytest.mark.gpu
BITS = 200


def two_pi() -> int:
    """2 pi times 2^BITS, by Machin's formula pi / 4 = 4 atan(1/5) - atan(1/239)."""
    one = 1 << (BITS + 20)

    def atan(n):
        total, t, k = 0, one // n, 0
        while t:
            total += (-1) ** k * (t // (2 * k + 1))
            t //= n * n
            k += 1
        return total

    return 8 * (4 * atan(5) - atan(239)) >> 20


def reduced(pos: int, freq: float, turn: int) -> float:
    """pos * freq modulo 2 pi, in [-pi, pi]."""
    num, den = freq.as_integer_ratio()
    r = (pos * num << BITS) // den % turn  # floors at 2^-200: far below fp64
    return (r - turn if 2 * r > turn else r) / (1 << BITS)


def test_reduced_angles():
    turn = two_pi()
    assert turn / (1 << BITS) == 2 * math.pi
    for pos in (1, 3, -3, 22, -355, 10 ** 6):  # fp64's own 2 pi is right to 2e-10 there
        assert reduced(pos, 1.0, turn) == pytest.approx(math.remainder(pos, 2 * math.pi), abs=2e-10)


@pytest.mark.parametrize("start", [-1500, 2 ** 29, 10 ** 10, 10 ** 12, 2 ** 45, -2 ** 50, 2 ** 53 - 1001])
def test_far_positions_keep_their_angle(start):
    T, nq, nkv, hd = 24, 2, 1, 128
    c = case(T, nq, nkv, hd, hd, 3, True, 16, start=start)
    run(c, nq, nkv, hd)
    K.check_device_errors(DEV)
    turn = two_pi()
    pos, freq, axes = c["positions"].tolist(), c["inv_freq"].tolist(), c["axes"].tolist()
    ang = torch.tensor([[reduced(pos[a][t], f, turn) for a, f in zip(axes, freq)] for t in range(T)], dtype=torch.float64)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]
    x = c["qkv"].double().cpu().view(T, nq + 2 * nkv, hd)[:, :nq + nkv]
    x[:, nq:] *= 0.75
    a, b = x.chunk(2, -1)
    ref = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    tol = 2.0 ** -8 * ref.abs() + 2.0 ** -20 * (a.abs() + b.abs()).repeat(1, 1, 2)
    block = c["key_cache"].shape[1]
    s = c["slots"]
    got = torch.cat([c["q_out"].view(T, nq, hd), c["key_cache"][s // block, s % block]], 1).double().cpu()
    off = (got - ref).abs()
    bad = int((~(off <= tol)).sum())
    assert bad == 0, f"{bad} of {off.numel()} off, worst by {float(off.max()):.3g}"
