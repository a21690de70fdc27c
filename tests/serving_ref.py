"""Plain 64-bit forms of the serving operators (clb200_qk_rope, clb200_attention, clb200_sample) and seeded inputs for them,
for the CPU and GPU tests. Everything here is numpy on the host."""
import numpy as np

# half a step of each type, relative to the value
HALF = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def positions(q_start, kv_len):
    """(row, sequence, position) of every row that belongs to a sequence."""
    out = []
    for s in range(len(kv_len)):
        a, z = q_start[s], q_start[s + 1]
        out += [(r, s, kv_len[s] - (z - r)) for r in range(a, z)]
    return out


def qk_rope(x, w, cs, norm, pairs, eps):
    """x [heads, hd] of one row, weights (or None), cs [hd] the row's cosines and sines -> (y, a bound on |terms of y|)."""
    H, D = x.shape
    if norm == 2:
        x = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * w
    elif norm == 1:
        x = x / np.sqrt((x * x).mean() + eps) * w.reshape(H, D)
    c, s = cs[:D // 2], cs[D // 2:]
    a, b = (x[:, 0::2], x[:, 1::2]) if pairs else (x[:, :D // 2], x[:, D // 2:])
    re, im, mag = a * c - b * s, a * s + b * c, np.abs(a) + np.abs(b)
    if pairs:
        return np.stack([re, im], 2).reshape(H, D), np.repeat(mag, 2, 1)
    return np.concatenate([re, im], 1), np.concatenate([mag, mag], 1)


def attention(q, k, v, pos, scale, window, sinks):
    """One row: q [H, hd], k and v [n, KV, hd] (the sequence's cache), pos -> (out, sum p |v|, sum |v| over visible, largest
    scale * sum |q k| over visible)."""
    H, D = q.shape
    KV = k.shape[1]
    j = np.arange(len(k))
    see = j <= pos
    if window > 0:
        see &= (j > pos - window) | (j < sinks)
    out, mag, flat, big = np.zeros((H, D)), np.zeros((H, D)), np.zeros((H, D)), np.zeros((H, 1))
    if see.any():
        for h in range(H):
            kk, vv = k[see, h // (H // KV)], v[see, h // (H // KV)]
            x = scale * (kk @ q[h])
            p = np.exp(x - x.max())
            p /= p.sum()
            out[h], mag[h], flat[h] = p @ vv, p @ np.abs(vv), np.abs(vv).sum(0)
            big[h] = scale * (np.abs(kk) @ np.abs(q[h])).max()
    return out, mag, flat, big


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row of logits -> (token, prob)."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if x.max() == -np.inf:
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 1.0
    M = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.exp((x - M) / float(temperature))
    w[x == -np.inf] = 0.0
    if M == np.inf:
        w[:] = 0.0
    w[x == M] = 1.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        c = np.cumsum(w[order])
        order = order[:min(int(np.searchsorted(c, max(float(top_p) * c[-1], 1e-300))) + 1, len(order))]
    if min_p > 0:
        order = order[w[order] >= min(float(min_p), 1.0)]
    order = np.sort(order)
    c = np.cumsum(w[order])
    u = min(max(float(u), 0.0), 1.0) if u == u else 0.0
    at = int(np.searchsorted(c, u * c[-1], side="right"))
    at = min(at, int(np.max(np.nonzero(w[order])[0])))
    return int(order[at]), float(w[order[at]] / c[-1])
