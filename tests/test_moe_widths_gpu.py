"""The mixture-of-experts layer at the widths of a model (hidden 2048, 8 of 256 experts of 512 and one that every token takes) on
one B200: at the sizes where its kernels change, and with experts of several row blocks. Formulas in 64 bits and tolerances
are those of test_moe_gpu.py; the routing weights add 2^-18 of the values, as there."""
import pytest
import torch

from multi_modal_parallelism_b200 import _lib
from multi_modal_parallelism_b200 import kernels as K
from tests.test_moe_gpu import BF, DEV, check_experts, experts_ref, gen, make, route_ref

pytestmark = pytest.mark.gpu
E, TOP, H, I = 256, 8, 2048, 512


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    torch.cuda.synchronize()
    K.check_device_errors(DEV)


def layer_case(T, n_experts=E, hidden=H, inter=I):
    x, wgu, wd, _, _, add = make(T, n_experts + 1, 1, hidden, inter, seed=T)
    return x, torch.randn(T, n_experts + 1, device=DEV, generator=gen(T + 1)).to(BF), wgu, wd, add


# 9 places a token: up to 7 tokens (63 places) one launch, 8 tokens are 72 places; the tensor-core kernels gather 128 rows a block up
# to 96 rows an expert (2741 tokens) and take sorted rows in blocks of 256 above; the shared expert has every token
@pytest.mark.parametrize("T", [1, 7, 8, 9, 33, 700, 2741, 2742])
def test_layer_with_a_shared_expert(T):
    x, l, wgu, wd, add = layer_case(T)
    out = K.moe_layer(x, l, wgu, wd, TOP, shared=True, addend=add)
    w, ids, _ = route_ref(l, E, TOP, True, True)
    ref, tol = experts_ref(x, wgu, wd, w, ids, add)
    tol = tol + 2.0 ** -18 * (ref.abs() + add.double().abs() + tol * 256)
    off = (out.double() - ref).abs()
    assert int((~(off <= tol)).sum()) == 0, f"worst {float((off / tol).max()):.3g} of the tolerance"


# (tokens, experts, places, hidden, intermediate): every token on the first experts, which so have several blocks of 128
# gathered rows (at most 96 rows an expert over all of them)
@pytest.mark.parametrize("T,n,k,hidden,inter", [(129, 64, 4, 2048, 1408), (1500, 64, 4, 1000, 264), (385, 256, 8, 2048, 512),
                                                (3000, 256, 8, 264, 520)])
def test_gathered_rows_of_experts_with_several_blocks(T, n, k, hidden, inter):
    assert T * k <= 96 * n
    a = make(T, n, k, hidden, inter, seed=T, skew=True, pad=2)
    check_experts(K.moe_experts(*a[:5], addend=a[5]), *a)
    a[4][:, 1:] = torch.randint(0, n, (T, k - 1), device=DEV, generator=gen(T)).int()  # one popular expert beside even ones
    check_experts(K.moe_experts(*a[:5], addend=a[5]), *a)


def kernel_nodes(call) -> int:
    """Kernels that the call launches: the kernel nodes of its captured graph."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    err, _, n = rt.cudaGraphGetNodes(raw)
    assert err == rt.cudaError_t.cudaSuccess
    err, nodes, n = rt.cudaGraphGetNodes(raw, n)
    assert err == rt.cudaError_t.cudaSuccess
    kinds = [rt.cudaGraphNodeGetType(node) for node in nodes[:n]]
    assert all(e == rt.cudaError_t.cudaSuccess for e, _ in kinds)
    return sum(t == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for _, t in kinds)


@pytest.mark.parametrize("T,n,k,hidden,inter", [
    (1, 16, 4, 1024, 64), (8, 16, 7, 1024, 64), (8, 16, 8, 1024, 64), (9, 16, 4, 1024, 64), (32, 16, 4, 1024, 64), (33, 16, 4, 1024, 64),
    (33, 16, 4, 1024, 520), (200, 16, 4, 1024, 64), (384, 16, 4, 1024, 64), (385, 16, 4, 1024, 64), (1000, 16, 4, 256, 128)])
def test_counted_launches_are_the_launched_kernels(T, n, k, hidden, inter):
    x, l, wgu, wd, add = layer_case(T, n, hidden, inter)
    out = torch.empty_like(x)
    ws = K.moe_workspace(T, k + 1, hidden, inter, n + 1, DEV)
    w, ids = K.moe_route(l, k, shared=True)
    for call in (lambda: K.moe_layer(x, l, wgu, wd, k, shared=True, addend=add, out=out, workspace=ws),
                 lambda: K.moe_experts(x, wgu, wd, w, ids, addend=add, out=out, workspace=ws)):
        call()
        torch.cuda.synchronize()
        before = _lib.LAUNCHES[0]
        launched = kernel_nodes(call)
        assert _lib.LAUNCHES[0] - before == launched
