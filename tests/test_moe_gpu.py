"""The mixture-of-experts kernels (kernels.moe_route, moe_experts, moe_layer) on one B200 against the formulas in 64 bits.

Tolerances. Routing: the chosen experts are exact; a weight exp(l - max) / Z has the rounding of l - max (2^-24 of it, an
absolute error of the exponent), expf's 2 units, the sum's and the division's: (|l - max| + E + 16) 2^-23 relative.
Products, element by element: h is rounded to bf16 and so is the result, half a step (2^-8) of each, h's carried through
|Wd|; every fp32 sum of n products errs by at most n 2^-24 of the sum of their magnitudes, and silu by 2^-18 of its value
(exp and divide of a few units each, the exponent's own rounding for |g| up to 32)."""
import math

import pytest
import torch

from multi_modal_parallelism_b200 import kernels as K
from multi_modal_parallelism_b200._lib import MmpError

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF = torch.bfloat16
INF = math.inf


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    torch.cuda.synchronize()
    K.check_device_errors(DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------------------ routing
def route_ref(logits, E, top_k, renorm, shared):
    l = logits[:, :E].double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -INF), l).clamp(max=torch.finfo(torch.float32).max)
    v, i = torch.sort(l, dim=1, descending=True, stable=True)
    top = v[:, :1]
    e = torch.where(torch.isinf(v), torch.zeros_like(v), torch.exp(v - torch.where(torch.isinf(top), torch.zeros_like(top), top)))
    z = (e[:, :top_k] if renorm else e).sum(1, keepdim=True)
    none = torch.isinf(v[:, :top_k])
    w = torch.where(none, torch.zeros_like(e[:, :top_k]), e[:, :top_k] / z)
    ids = torch.where(none, torch.full_like(i[:, :top_k], -1), i[:, :top_k])
    gap = torch.where(none, torch.zeros_like(w), (top - v[:, :top_k]).abs())
    if shared:
        w = torch.cat([w, torch.sigmoid(logits[:, E:].double())], 1)
        ids = torch.cat([ids, torch.full_like(ids[:, :1], E)], 1)
        gap = torch.cat([gap, logits[:, E:].double().abs().clamp(max=1e3)], 1)
    return w, ids.int(), gap


def check_route(logits, E, top_k, renorm, shared, got):
    w, ids, gap = route_ref(logits, E, top_k, renorm, shared)
    assert torch.equal(got[1], ids)
    tol = w * (gap + E + 16) * 2.0 ** -23 + 2.0 ** -126
    assert bool(((got[0].double() - w).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("T,E,top_k", [(1, 1, 1), (1, 8, 8), (3, 33, 5), (64, 256, 8), (65, 60, 4), (129, 257, 10), (1000, 160, 6),
                                       (31, 1024, 31)])
@pytest.mark.parametrize("renorm,shared", [(True, False), (False, True)])
def test_route(dtype, T, E, top_k, renorm, shared):
    l = (torch.randn(T, E + shared, device=DEV, generator=gen(E)) * 2).to(dtype)
    check_route(l, E, top_k, renorm, shared, K.moe_route(l, top_k, renormalize=renorm, shared=shared))


@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_route_ties_masks_and_non_finite_values(dtype):
    E, k = 40, 6
    l = torch.randn(12, E, device=DEV, generator=gen(1))
    l[0] = 0.0                                   # all equal: the first experts in order
    l[1] = -INF                                  # nothing left
    l[2] = -INF
    l[2, 37] = -3e38                             # one left, at nearly the type's lowest value
    l[3] = torch.finfo(dtype).min                # masks of the type's lowest value tie like any other
    l[4, ::2] = -INF
    l[5, 3] = INF                                # takes all
    l[6, [3, 30]] = INF                          # two of them share
    l[7] = math.nan
    l[8, 5:] = math.nan                          # fewer than k left
    l[9] = torch.tensor([0.0, -0.0] * (E // 2))  # the two zeros tie
    l[10] = torch.arange(E) * -200.0             # weights underflow to zero, the order holds
    l = l.to(dtype)
    for renorm in (True, False):
        w, ids = K.moe_route(l, k, renormalize=renorm)
        check_route(l, E, k, renorm, False, (w, ids))
        assert ids[1].tolist() == [-1] * k and w[1].tolist() == [0.0] * k
        assert ids[8].tolist()[5:] == [-1] and bool(torch.isfinite(w).all())
        assert ids[9].tolist() == list(range(k))


def test_route_strided_logits_and_given_outputs():
    wide = torch.randn(50, 100, device=DEV, generator=gen(3)).to(BF)
    l = wide[:, 7:71]
    w, ids = torch.full((50, 4), 9.0, device=DEV), torch.full((50, 4), 9, dtype=torch.int32, device=DEV)
    got = K.moe_route(l, 4, weights=w, ids=ids)
    assert got[0] is w and got[1] is ids
    check_route(l, 64, 4, True, False, got)


# ------------------------------------------------------------------------------------------------ products
def experts_ref(x, wgu, wd, weights, ids, addend):
    """(out, tolerance) in 64 bits, expert by expert."""
    T, H = x.shape
    E, I = wd.shape[0], wd.shape[2]
    u24 = 2.0 ** -24
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device) if addend is None else addend.double()
    mag = out.abs()                     # magnitudes of the sum over places
    err = torch.zeros_like(out)         # error before the last rounding
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe, w = x[t].double(), weights[t, j].double()[:, None]
        wg, wu, d = wgu[e, :I].double(), wgu[e, I:].double(), wd[e].double()
        g, u = xe @ wg.T, xe @ wu.T
        s = g * torch.sigmoid(g)
        h = s * u
        dg, du = (H * u24) * (xe.abs() @ wg.abs().T), (H * u24) * (xe.abs() @ wu.abs().T)
        dh = 1.1 * dg * (u.abs() + du) + s.abs() * du + 2.0 ** -18 * h.abs()
        dh = dh + 2.0 ** -8 * (h.abs() + dh)
        y, ya = h @ d.T, (h.abs() + dh) @ d.abs().T
        out.index_add_(0, t, w * y)
        mag.index_add_(0, t, w.abs() * ya)
        err.index_add_(0, t, w.abs() * (dh @ d.abs().T + I * u24 * ya))
    err = err + (ids.shape[1] + 2) * 2 * u24 * mag
    return out, err + 2.0 ** -8 * (out.abs() + err) + 2.0 ** -130


def make(T, E, k, H, I, seed=0, skew=False, pad=0):
    g = gen(seed)
    x = torch.randn(T, H, device=DEV, generator=g).to(BF)
    wgu = (torch.randn(E, 2 * I, H, device=DEV, generator=g) / math.sqrt(H)).to(BF)
    wd = (torch.randn(E, H, I, device=DEV, generator=g) / math.sqrt(I)).to(BF)
    v, ids = torch.randn(T, E, device=DEV, generator=g).topk(k, 1)
    if skew:
        ids = torch.arange(k, device=DEV).expand(T, k).contiguous()
    ids = ids.int()
    if pad:
        ids[-pad:] = -1
    return x, wgu, wd, torch.softmax(v, 1), ids, torch.randn(T, H, device=DEV, generator=g).to(BF)


def check_experts(got, x, wgu, wd, weights, ids, addend):
    ref, tol = experts_ref(x, wgu, wd, weights, ids, addend)
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.3g} of the tolerance"


# (tokens, experts, places, hidden, intermediate): one launch for up to 8 tokens, the few-token kernels while places times
# intermediate is small, the tensor-core ones else; small sizes of either path are in both lists
FEW = [(1, 1, 1, 8, 8), (1, 4, 1, 16, 8), (1, 8, 2, 256, 64), (2, 64, 8, 2048, 512), (5, 16, 4, 264, 72), (7, 30, 9, 2408, 136),
       (8, 8, 8, 128, 64), (9, 4, 2, 520, 40), (17, 2, 1, 128, 640), (40, 60, 4, 1000, 120), (384, 1000, 4, 64, 24),
       (30, 16, 2, 4104, 264), (300, 300, 4, 2400, 8), (33, 8, 2, 512, 136), (64, 60, 4, 104, 24), (100, 40, 3, 264, 72),
       (20, 8, 2, 4808, 40), (1, 1024, 32, 72, 8),
       (64, 60, 2, 2048, 512), (100, 60, 2, 2408, 136), (64, 8, 2, 2048, 264), (50, 8, 2, 4808, 40), (100, 8, 4, 2048, 72)]
MANY = [(64, 8, 2, 4104, 264), (170, 12, 9, 96, 1032), (1537, 3, 1, 64, 24), (777, 5, 3, 8, 8), (600, 8, 4, 264, 72), (900, 16, 2, 1024, 200), (2000, 64, 8, 136, 64),
        (257, 16, 8, 2048, 512), (4097, 2, 1, 128, 328), (513, 1, 4, 72, 128), (1024, 300, 6, 64, 40)]


@pytest.mark.parametrize("T,E,k,H,I", FEW)
def test_experts_few_tokens(T, E, k, H, I):
    a = make(T, E, min(k, E), H, I, seed=T)
    check_experts(K.moe_experts(*a[:5], addend=a[5]), *a)


@pytest.mark.parametrize("T,E,k,H,I", MANY)
def test_experts_many_tokens(T, E, k, H, I):
    a = make(T, E, min(k, E), H, I, seed=T)
    if k > E:  # the same expert several times for a token
        a = (*a[:3], torch.rand(T, k, device=DEV, generator=gen(1)), torch.zeros(T, k, dtype=torch.int32, device=DEV), a[5])
    check_experts(K.moe_experts(*a[:5], addend=a[5]), *a)


@pytest.mark.parametrize("T,E,k,H,I", [(20, 16, 2, 512, 96), (100, 16, 2, 512, 96), (1000, 16, 2, 512, 96)])
def test_experts_all_tokens_on_the_same_experts(T, E, k, H, I):
    a = make(T, E, k, H, I, skew=True)
    check_experts(K.moe_experts(*a[:5], addend=a[5]), *a)


@pytest.mark.parametrize("T", [40, 200, 1100])
def test_experts_without_addend_and_rows_without_experts(T):
    a = make(T, 16, 4, 1024, 64, pad=7)
    a[4][3] = -1           # a whole row
    a[4][5, 1:] = -1       # some of its places
    a[4][6, 1] = a[4][6, 0]  # the same expert twice
    a[3][3] = math.nan     # weights of empty places are not used
    out = K.moe_experts(*a[:5])
    check_experts(out, *a[:5], None)
    assert not bool(out[3].any()) and not bool(out[-7:].any())
    out = K.moe_experts(*a[:5], addend=a[5])
    assert torch.equal(out[3], a[5][3]) and torch.equal(out[-7:], a[5][-7:])


@pytest.mark.parametrize("T", [3, 20, 100, 1000])
def test_experts_no_places_at_all(T):
    a = make(T, 8, 2, 512, 64)
    a[4].fill_(-1)
    assert torch.equal(K.moe_experts(*a[:5], addend=a[5]), a[5])


@pytest.mark.parametrize("T", [4, 10, 100, 1000])
def test_experts_index_out_of_range_is_reported_and_adds_nothing(T):
    a = make(T, 8, 2, 512, 64)
    ids = a[4].clone()
    a[4][1, 0] = 8
    ids[1, 0] = -1
    out = K.moe_experts(*a[:5], addend=a[5])
    with pytest.raises(MmpError, match="index out of range"):
        K.check_device_errors(DEV)
    check_experts(out, a[0], a[1], a[2], a[3], ids, a[5])


@pytest.mark.parametrize("T", [10, 100, 1000])
def test_experts_strided_rows_and_out_over_the_addend(T):
    E, k, H, I = 8, 2, 520, 72
    a = make(T, E, k, H, I)
    x = torch.zeros(T, H + 24, dtype=BF, device=DEV)[:, 8:8 + H].copy_(a[0])
    wgu = torch.zeros(E, 2 * I + 3, H + 8, dtype=BF, device=DEV)[:, :2 * I, :H].copy_(a[1])
    wd = torch.zeros(E, H + 1, I + 16, dtype=BF, device=DEV)[:, :H, 8:8 + I].copy_(a[2])
    weights = torch.zeros(T, k + 3, device=DEV)[:, 1:1 + k].copy_(a[3])
    ids = torch.zeros(T, k + 5, dtype=torch.int32, device=DEV)[:, 2:2 + k].copy_(a[4])
    guard = torch.full((T, H + 16), 7.0, dtype=BF, device=DEV)
    out = guard[:, 8:8 + H].copy_(a[5])
    assert K.moe_experts(x, wgu, wd, weights, ids, out=out, addend=out) is out
    check_experts(out, *a)
    assert bool((guard[:, :8] == 7).all()) and bool((guard[:, 8 + H:] == 7).all())


@pytest.mark.parametrize("T", [24, 60, 1000])
def test_experts_non_finite_token_stays_in_its_row(T):
    a = make(T, 4, 2, 512, 64)
    clean = K.moe_experts(*a[:5], addend=a[5])
    a[0][5, 3] = math.nan
    a[0][7, 3] = INF
    out = K.moe_experts(*a[:5], addend=a[5])
    keep = torch.ones(T, dtype=torch.bool, device=DEV)
    keep[[5, 7]] = False
    assert torch.equal(out[keep], clean[keep]) and bool(torch.isnan(out[5]).all())


@pytest.mark.parametrize("T", [16, 100, 1000])
def test_experts_same_bits_every_time(T):
    a = make(T, 16, 4, 1024, 128)
    first = K.moe_experts(*a[:5], addend=a[5])
    for _ in range(5):
        assert torch.equal(K.moe_experts(*a[:5], addend=a[5]), first)


def test_empty_batch():
    a = make(4, 8, 2, 128, 64)
    out = K.moe_experts(a[0][:0], a[1], a[2], a[3][:0], a[4][:0])
    assert out.shape == (0, 128)
    assert K.moe_layer(a[0][:0], torch.zeros(0, 8, device=DEV), a[1], a[2], 2).shape == (0, 128)
    w, ids = K.moe_route(torch.zeros(0, 8, device=DEV), 2)
    assert w.shape == ids.shape == (0, 2)


# ------------------------------------------------------------------------------------------------ layer
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("T,E,k,H,I,shared", [(1, 16, 4, 256, 64, True), (7, 256, 8, 512, 128, True), (64, 40, 6, 264, 72, False),
                                              (200, 8, 2, 128, 64, True), (700, 16, 4, 256, 128, True), (1700, 30, 1, 64, 32, False),
                                              (20, 16, 4, 1024, 64, True), (60, 16, 4, 2048, 64, True)])
def test_layer_is_route_and_experts(dtype, T, E, k, H, I, shared):
    n = E + shared
    x, wgu, wd, _, _, add = make(T, n, 1, H, I, seed=E)
    l = torch.randn(T, n, device=DEV, generator=gen(9)).to(dtype)
    l[0, 1:E] = -INF  # a token with one expert left
    out = K.moe_layer(x, l, wgu, wd, k, shared=shared, addend=add)
    w, ids, _ = route_ref(l, E, k, True, shared)
    ref, tol = experts_ref(x, wgu, wd, w, ids, add)
    # routing weights to 2^-18 relative: far below the roundings of the products
    tol = tol + 2.0 ** -18 * (ref.abs() + add.double().abs() + tol * 256)
    assert bool(((out.double() - ref).abs() <= tol).all())
    w2, ids2 = K.moe_route(l, k, shared=shared)
    assert torch.equal(K.moe_experts(x, wgu, wd, w2, ids2, addend=add), out)


@pytest.mark.parametrize("T", [8, 40, 200, 600])
def test_layer_captured_and_replayed_on_new_inputs(T):
    E, k, H, I = 16, 4, 1024, 64
    x, wgu, wd, _, _, add = make(T, E + 1, 1, H, I)
    l = torch.randn(T, E + 1, device=DEV, generator=gen(2)).to(BF)
    out = torch.empty(T, H, dtype=BF, device=DEV)
    ws = K.moe_workspace(T, k + 1, H, I, E + 1, DEV)
    call = lambda: K.moe_layer(x, l, wgu, wd, k, out=out, shared=True, addend=add, workspace=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in (5, 6):
        x.copy_(torch.randn(T, H, device=DEV, generator=gen(seed)))
        l.copy_(torch.randn(T, E + 1, device=DEV, generator=gen(seed + 10)))
        graph.replay()
        replayed = out.clone()
        assert torch.equal(replayed, K.moe_layer(x, l, wgu, wd, k, shared=True, addend=add))


@pytest.mark.parametrize("T", [8, 20, 100, 600])
def test_two_streams_at_once(T):
    """Calls on two streams overlap; each has scratch of its own when none is given."""
    a, b = make(T, 16, 4, 1024, 128, seed=1), make(T, 16, 4, 1024, 128, seed=2)
    want = [K.moe_experts(*q[:5], addend=q[5]) for q in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, q in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(K.moe_experts(*q[:5], addend=q[5]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T", [5, 40, 200, 700])
def test_layer_rows_whose_mask_leaves_nothing(T, renorm):
    """A token with every expert masked gets the addend alone, with the shared expert that one's share."""
    E, k, H, I = 16, 4, 1024, 64
    x, wgu, wd, _, _, add = make(T, E + 1, 1, H, I)
    l = torch.randn(T, E + 1, device=DEV, generator=gen(4)).to(BF)
    l[[1, T - 1], :E] = -INF
    out = K.moe_layer(x, l[:, :E], wgu[:E], wd[:E], k, renormalize=renorm, addend=add)
    assert torch.equal(out[[1, T - 1]], add[[1, T - 1]])
    w, ids = K.moe_route(l[:, :E], k, renormalize=renorm)
    assert ids[1].tolist() == [-1] * k
    assert torch.equal(out, K.moe_experts(x, wgu[:E], wd[:E], w, ids, addend=add))
    check_experts(out, x, wgu[:E], wd[:E], w, ids, add)
    out = K.moe_layer(x, l, wgu, wd, k, renormalize=renorm, shared=True, addend=add)
    w, ids = K.moe_route(l, k, renormalize=renorm, shared=True)
    assert ids[1].tolist() == [-1] * k + [E]
    check_experts(out, x, wgu, wd, w, ids, add)


def test_one_scratch_for_calls_of_every_path_in_a_row():
    """Calls that follow one another on a stream share one scratch, sized for the largest; none is waited for."""
    E, k, H, I = 16, 4, 2048, 128
    batches = [3, 900, 40, 8, 1500, 200, 1, 64]
    data = [make(T, E, k, H, I, seed=T) for T in batches]
    want = [K.moe_experts(*a[:5], addend=a[5]) for a in data]
    ws = K.moe_workspace(max(batches), k, H, I, E, DEV)
    torch.cuda.synchronize()
    for _ in range(5):
        got = [K.moe_experts(*a[:5], addend=a[5], workspace=ws) for a in data]
    for g, w in zip(got, want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("T", [8, 40, 200, 600])
def test_two_captured_graphs_with_a_scratch_each(T):
    E, k, H, I = 16, 4, 1024, 64
    data = [make(T, E, k, H, I, seed=s) for s in (1, 2)]
    want = [K.moe_experts(*a[:5], addend=a[5]) for a in data]
    graphs, outs, streams = [], [], [torch.cuda.Stream(DEV) for _ in data]
    for a in data:
        ws, out = K.moe_workspace(T, k, H, I, E, DEV), torch.empty(T, H, dtype=BF, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(4):
                K.moe_experts(*a[:5], addend=a[5], out=out, workspace=ws)
        graphs.append(graph)
        outs.append((out, ws))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (out, _), w in zip(outs, want):
        assert torch.equal(out, w)


def test_chained_layers_read_what_the_one_before_wrote():
    """Each call's output is the next one's input, on every path, without a wait: the same bits as with one."""
    E, k, H, I = 16, 4, 1024, 64
    for T in (8, 40, 200, 600):
        x, wgu, wd, w, ids, _ = make(T, E, k, H, I, seed=T)
        y = x
        for _ in range(6):
            y = K.moe_experts(y, wgu, wd, w, ids, addend=y)
        z = x
        for _ in range(6):
            torch.cuda.synchronize()
            z = K.moe_experts(z, wgu, wd, w, ids, addend=z)
        assert torch.equal(y, z)
