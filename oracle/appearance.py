"""64-bit restatements of the learned-appearance operators (layer norm, gated
feed-forward block, counter-based dropout), from their formulas."""
from __future__ import annotations

import numpy as np
import torch


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias; torch tensors, differentiable."""
    z = x - x.mean(-1, keepdim=True)
    z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
    z = z if weight is None else z * weight
    return z if bias is None else z + bias


def layer_norm_grads(x, weight, eps, v_y):
    """(v_x, v_weight, v_bias) from the closed formulas."""
    c = x.shape[-1]
    d = x - x.mean(-1, keepdim=True)
    std = torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    z = d / std
    v = v_y if weight is None else v_y * weight
    v_x = (v - v.sum(-1, keepdim=True) / c - z * (v * z).sum(-1, keepdim=True) / c) / std
    return v_x, (v_y * z).sum(0), v_y.sum(0)


def silu(g):
    return g / (1 + torch.exp(-g))


def silu_slope(g):
    s = 1 / (1 + torch.exp(-g))
    return s + g * s * (1 - s)


def gated_feed_forward(x, w_gate, w_up, w_down):
    return (silu(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T


def gated_feed_forward_grads(x, w_gate, w_up, w_down, v_y):
    """(v_x, v_w_gate, v_w_up, v_w_down) from the closed formulas."""
    g, u = x @ w_gate.T, x @ w_up.T
    v_h = v_y @ w_down
    v_u, v_g = v_h * silu(g), v_h * u * silu_slope(g)
    return v_g @ w_gate + v_u @ w_up, v_g.T @ x, v_u.T @ x, v_y.T @ (silu(g) * u)


def philox4x32_10(counter, key):
    """Philox4x32-10 (Salmon et al. 2011): four uint64 arrays of 32-bit
    counter words and two key words -> four arrays of 32-bit words."""
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & mask,
             (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def dropout_keep(n, c, p, seed, offset=0, ids=None, per_row=False):
    """Bool [n, c]: which values are kept."""
    ids = np.arange(n, dtype=np.int64) if ids is None else np.asarray(ids, dtype=np.int64)
    ids = ids.astype(np.uint64)[:, None]
    col = np.arange(1 if per_row else c, dtype=np.uint64)[None, :]
    shape = (n, col.shape[1])
    words = philox4x32_10([np.broadcast_to(v, shape) for v in
                           (ids & np.uint64(0xFFFFFFFF), ids >> np.uint64(32), col >> np.uint64(2),
                            np.full((1, 1), offset & 0xFFFFFFFF, dtype=np.uint64))],
                          (seed & 0xFFFFFFFF, seed >> 32))
    words = np.choose((col & np.uint64(3)).astype(np.int64) + np.zeros(shape, dtype=np.int64), words)
    keep = words >= np.uint64(int(p * 2 ** 32))
    return np.broadcast_to(keep, (n, c)).copy()
