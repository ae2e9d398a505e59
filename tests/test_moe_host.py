"""Refusals of the mixture-of-experts and several-axis rotary entry points, on a machine without a GPU: the wrappers and the
C library check their arguments before any CUDA call. The wrappers run with CPU tensors and only their device assertion
relaxed; a call that reached a launch would not raise ValueError."""
import pytest
import torch

from multi_modal_parallelism_b200 import _lib
from multi_modal_parallelism_b200 import kernels as K
from multi_modal_parallelism_b200.state import alloc_kv

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
T, E, k, H, I = 4, 8, 2, 64, 32


@pytest.fixture
def cpu(monkeypatch):
    monkeypatch.setattr(K, "_cuda", lambda *a, **kw: None)
    monkeypatch.setattr(K, "_stream", lambda t: None)
    monkeypatch.setattr(K, "error_word", lambda dev: torch.zeros(1, dtype=I32))


def experts(**kw):
    a = dict(x=torch.zeros(T, H, dtype=BF), w_gate_up=torch.zeros(E, 2 * I, H, dtype=BF), w_down=torch.zeros(E, H, I, dtype=BF),
             weights=torch.zeros(T, k), ids=torch.zeros(T, k, dtype=I32))
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    off = -ws.data_ptr() % 256
    a["workspace"] = ws[off:]
    a.update(kw)
    return a


def test_cuda_tensors_are_required():
    with pytest.raises(ValueError, match="CUDA device"):
        K.moe_experts(**experts())
    with pytest.raises(ValueError, match="CUDA device"):
        K.moe_route(torch.zeros(T, E), k)
    with pytest.raises(ValueError, match="CUDA device"):
        K.moe_layer(torch.zeros(T, H, dtype=BF), torch.zeros(T, E), torch.zeros(E, 2 * I, H, dtype=BF), torch.zeros(E, H, I, dtype=BF), k)


@pytest.mark.parametrize("bad", [
    dict(x=torch.zeros(T, H)),                                             # type
    dict(weights=torch.zeros(T, k, dtype=BF)),
    dict(ids=torch.zeros(T, k, dtype=torch.int64)),
    dict(ids=torch.zeros(T, k + 1, dtype=I32)),                            # shapes that disagree
    dict(ids=torch.zeros(T + 1, k, dtype=I32), weights=torch.zeros(T + 1, k)),
    dict(w_down=torch.zeros(E, H, I + 8, dtype=BF)),
    dict(w_gate_up=torch.zeros(E + 1, 2 * I, H, dtype=BF)),
    dict(out=torch.zeros(T, H + 8, dtype=BF)),
    dict(addend=torch.zeros(T - 1, H, dtype=BF)),
    dict(out=torch.zeros(H, T, dtype=BF).t()),                             # rows not contiguous
    dict(w_down=torch.zeros(E, I, H, dtype=BF).transpose(1, 2)),
    dict(x=torch.zeros(T, 2 * H + 1, dtype=BF)[:, 1:H + 1]),               # rows not aligned
    dict(x=torch.zeros(T, H + 4, dtype=BF)[:, :H]),
    dict(weights=torch.zeros(T, 33), ids=torch.zeros(T, 33, dtype=I32)),   # too many places
    dict(weights=torch.zeros(T, 0), ids=torch.zeros(T, 0, dtype=I32)),
    dict(workspace=torch.zeros(16, dtype=torch.uint8)),                    # scratch too small, then misaligned
    dict(workspace=experts()["workspace"][8:]),
    dict(x=torch.zeros(1, H, dtype=BF).expand(T, H)),                      # rows that overlap
    dict(out=torch.zeros(1, H, dtype=BF).expand(T, H)),
])
def test_experts_refuses(cpu, bad):
    with pytest.raises(ValueError):
        K.moe_experts(**experts(**bad))


@pytest.mark.parametrize("H_,I_", [(60, 32), (64, 36), (64, 0)])
def test_experts_refuses_widths(cpu, H_, I_):
    with pytest.raises(ValueError):
        K.moe_experts(**experts(x=torch.zeros(T, H_, dtype=BF), w_gate_up=torch.zeros(E, 2 * I_, H_, dtype=BF),
                                w_down=torch.zeros(E, H_, I_, dtype=BF)))


def test_experts_refuses_too_many_experts(cpu):
    n = 1025
    with pytest.raises(ValueError):
        K.moe_experts(**experts(w_gate_up=torch.zeros(n, 16, 8, dtype=BF), w_down=torch.zeros(n, 8, 8, dtype=BF),
                                x=torch.zeros(T, 8, dtype=BF)))


@pytest.mark.parametrize("logits,top_k,kw", [
    (torch.zeros(T, E), 0, {}), (torch.zeros(T, E), E + 1, {}), (torch.zeros(T, E), E, {"shared": True}),
    (torch.zeros(T, 1025), 2, {}), (torch.zeros(T, 64), 33, {}), (torch.zeros(T, 64), 32, {"shared": True}),
    (torch.zeros(T, E, dtype=torch.float16), k, {}), (torch.zeros(E, T).t(), k, {}), (torch.zeros(1, E).expand(T, E), k, {}),
    (torch.zeros(T, E), k, {"weights": torch.zeros(T, k + 1)}), (torch.zeros(T, E), k, {"ids": torch.zeros(T, k, dtype=torch.int64)}),
    (torch.zeros(T, E), k, {"weights": torch.zeros(T, 2 * k)[:, ::2]})])
def test_route_refuses(cpu, logits, top_k, kw):
    with pytest.raises(ValueError):
        K.moe_route(logits, top_k, **kw)


@pytest.mark.parametrize("logits,top_k,shared", [(torch.zeros(T, E + 1), k, True), (torch.zeros(T + 1, E), k, False),
                                                 (torch.zeros(T, E), E, True), (torch.zeros(T, E), 0, False)])
def test_layer_refuses(cpu, logits, top_k, shared):
    a = experts()
    with pytest.raises(ValueError):
        K.moe_layer(a["x"], logits, a["w_gate_up"], a["w_down"], top_k, shared=shared, workspace=a["workspace"])


def test_empty_batches_return_without_a_launch(cpu):
    a = experts(x=torch.zeros(0, H, dtype=BF), weights=torch.zeros(0, k), ids=torch.zeros(0, k, dtype=I32))
    assert K.moe_experts(**a).shape == (0, H)
    assert K.moe_layer(a["x"], torch.zeros(0, E), a["w_gate_up"], a["w_down"], k).shape == (0, H)
    assert K.moe_route(torch.zeros(0, E), k)[1].shape == (0, k)


def test_workspace_size_grows_with_the_request():
    size = lambda *a: _lib.lib().mmp_moe_workspace_size(*a)  # noqa: E731
    assert size(0, 2, 64, 32, 8) == 0
    assert 0 < size(4, 2, 64, 32, 8) <= size(5, 2, 64, 32, 8)
    # scratch of a larger request serves a smaller one, whichever kernels take either
    for rest in ((2, 64, 32, 8), (8, 2048, 512, 257), (1, 8, 8, 3), (32, 8, 8, 1024), (2, 4096, 7168, 8)):
        got = [size(T, *rest) for T in range(1, 2200)]
        assert all(x <= y for x, y in zip(got, got[1:])), rest
    R = 1000 * 2  # a large request holds the fp32 results and the bf16 intermediate rows
    assert size(1000, 2, 64, 32, 8) >= R * (64 * 4 + 32 * 2)
    # 64-bit sizes: 2^25 places of 8192 columns
    assert size(1 << 22, 8, 8192, 1024, 64) >= (1 << 25) * (8192 * 4 + 1024 * 2)


# ------------------------------------------------------------------------------------------------ rotary
def mrope(**kw):
    nq, nkv, hd = 4, 2, 64
    _, kc, vc, _ = alloc_kv(2, 16, nkv, hd, torch.device("cpu"))
    a = dict(qkv=torch.zeros(T, (nq + 2 * nkv) * hd, dtype=BF), nq=nq, nkv=nkv, head_dim=hd,
             positions=torch.zeros(3, T, dtype=torch.int64), inv_freq=torch.zeros(32), axes=torch.zeros(32, dtype=I32), key_mult=1.0,
             q_out=torch.zeros(T, nq * hd, dtype=BF), key_cache=kc, value_cache=vc, slot_mapping=torch.zeros(T, dtype=torch.int64))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(qkv=torch.zeros(T, 8 * 64)), dict(qkv=torch.zeros(T, 9 * 64, dtype=BF)), dict(positions=torch.zeros(T, dtype=torch.int64)),
    dict(positions=torch.zeros(3, T + 1, dtype=torch.int64)), dict(positions=torch.zeros(3, T, dtype=I32)),
    dict(positions=torch.zeros(T, 3, dtype=torch.int64).t()), dict(inv_freq=torch.zeros(33)), dict(axes=torch.zeros(32, dtype=torch.int64)),
    dict(inv_freq=torch.zeros(33), axes=torch.zeros(33, dtype=I32)), dict(inv_freq=torch.zeros(0), axes=torch.zeros(0, dtype=I32)),
    dict(inv_freq=torch.zeros(64)[::2]), dict(q_out=torch.zeros(T, 4 * 64 + 8, dtype=BF)), dict(slot_mapping=torch.zeros(T, dtype=I32)),
    dict(slot_mapping=torch.zeros(T + 1, dtype=torch.int64)), dict(key_cache=torch.zeros(2, 16, 2, 64, dtype=BF)),
    dict(key_cache=torch.zeros(2, 16, 4, 64, dtype=BF), value_cache=torch.zeros(2, 16, 4, 64, dtype=BF)),
    dict(key_cache=torch.zeros(2, 16, 2, 64), value_cache=torch.zeros(2, 16, 2, 64)),
    dict(positions=torch.zeros(0, T, dtype=torch.int64)), dict(q_out=torch.zeros(1, 4 * 64, dtype=BF).expand(T, 256)),
])
def test_mrope_refuses(cpu, bad):
    with pytest.raises(ValueError):
        K.qkv_mrope_kv_write(**mrope(**bad))


def test_mrope_cuda_tensors_are_required():
    with pytest.raises(ValueError, match="CUDA device"):
        K.qkv_mrope_kv_write(**mrope())


def test_rope_axes():
    dev = torch.device("cpu")
    assert K.rope_axes([2, 1, 1], False, dev).tolist() == [0, 0, 1, 2]
    assert K.rope_axes([4, 2, 2], True, dev).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert K.rope_axes([3], True, dev).tolist() == [0, 0, 0]
    a = K.rope_axes([24, 20, 20], True, dev)
    assert [int((a == i).sum()) for i in range(3)] == [24, 20, 20] and a.dtype == I32
    for bad in ([], [0, 0], [2, -1], ):
        with pytest.raises(ValueError):
            K.rope_axes(bad, False, dev)
    with pytest.raises(ValueError):
        K.rope_axes([1, 4, 4], True, dev)  # pairs of the other axes run out of places


@pytest.mark.parametrize("T,places,H,I,E,launches", [
    (1, 9, 2048, 512, 257, (1, 1)),         # one launch
    (30, 4, 2048, 64, 16, (3, 3)),          # plan (with the routing of few tokens), up, down
    (60, 4, 2048, 64, 16, (3, 4)),
    (200, 4, 2048, 512, 16, (4, 5)),        # plan, up, down, sum
    (2000, 4, 2048, 512, 16, (5, 6)),       # plan, sorted rows, up, down, sum
])
def test_launches_and_scratch(T, places, H, I, E, launches):
    lib = _lib.lib()
    assert tuple(lib.mmp_moe_launches(T, places, H, I, E, r) for r in (0, 1)) == launches
    # the scratch of a request serves every smaller one
    sizes = [lib.mmp_moe_workspace_size(t, places, H, I, E) for t in range(1, T + 1)]
    assert sizes == sorted(sizes)
