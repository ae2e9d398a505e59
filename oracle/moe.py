"""numpy fp32 mixture-of-experts MLP and several-axis rotary angles of the Gated DeltaNet stack: test infrastructure only.

The reference describes this model family (`configs/qwen35_35b_a3b.yaml:1-22`) and has no implementation of it: parity
unpinned; the formulas are the operators' own definitions.
"""
from __future__ import annotations

import numpy as np

from .hybrid_layer import F32, gemm, silu


def moe_route(logits: np.ndarray, top_k: int) -> tuple[np.ndarray, np.ndarray]:
    """The top_k largest of each row (ties to the lowest index) and their softmax."""
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    v = np.take_along_axis(logits, ids, 1)
    w = np.exp(v - v[:, :1])
    return ids, (w / w.sum(1, keepdims=True)).astype(F32)


def moe_mlp(w: dict, d, y: np.ndarray, logits: np.ndarray | None = None) -> np.ndarray:
    """y [T, H] through the routed experts and, with its weights there, the shared one behind its sigmoid gate. logits
    (default y times the router) [T, experts (+ 1)]."""
    gu, down = w["mlp.experts.gate_up_proj"], w["mlp.experts.down_proj"]
    E, n = down.shape[0], down.shape[2]
    shared = "mlp.shared_expert_gate.weight" in w
    if logits is None:
        logits = gemm(y, w["mlp.gate.weight"])
        if shared:
            logits = np.concatenate([logits, gemm(y, w["mlp.shared_expert_gate.weight"])], 1)
    ids, wt = moe_route(logits[:, :E], d.top_k)
    out = np.zeros_like(y, F32)
    for e in range(E):
        t, k = np.nonzero(ids == e)
        if t.size:
            h = silu(gemm(y[t], gu[e, :n])) * gemm(y[t], gu[e, n:])
            out[t] += wt[t, k][:, None] * gemm(h, down[e])
    if shared:
        h = silu(gemm(y, w["mlp.shared_expert.gate_proj.weight"])) * gemm(y, w["mlp.shared_expert.up_proj.weight"])
        out += gemm(h, w["mlp.shared_expert.down_proj.weight"]) / (F32(1) + np.exp(-logits[:, E:]))
    return out


def axis_cos_sin(positions: np.ndarray, sections, interleaved: bool, rotary_dim: int, theta: float):
    """positions [axes, L] -> cos, sin [L, rotary_dim / 2]: pair i turns with its axis' position; interleaved: axis i mod n
    while i < n * sections[i mod n], axis 0 otherwise; else in blocks of sections[a] pairs."""
    n, half = len(sections), rotary_dim // 2
    if interleaved:
        ax = np.array([i % n if i < n * sections[i % n] else 0 for i in range(half)])
    else:
        ax = np.repeat(np.arange(n), sections)
    inv = F32(1.0) / (F32(theta) ** (np.arange(0, rotary_dim, 2, dtype=F32) / F32(rotary_dim)))
    ang = np.asarray(positions, np.float64)[ax].T * inv.astype(np.float64)
    return np.cos(ang).astype(F32), np.sin(ang).astype(F32)


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray) -> np.ndarray:
    """x [L, heads, hd]: dims (i, i + half) of the first 2 * half turn, the others pass."""
    h = cos.shape[1]
    a, b, c, s = x[..., :h], x[..., h:2 * h], cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)
