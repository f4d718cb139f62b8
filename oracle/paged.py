"""The operators over a paged cache and the row sampler, from their definitions: numpy, 64 bits, one sequence, head and
row at a time.  Tensors of 16-bit types come as float64 arrays of their values."""
from __future__ import annotations

import math

import numpy as np


def rows_of(pages, table, length):
    """``[length, KH, D]`` and which of them have a page, from pages ``[n, KH, P, D]`` and one table row."""
    n, kh, p, d = pages.shape
    length = min(max(int(length), 0), len(table) * p)
    out = np.zeros((length, kh, d))
    there = np.zeros(length, bool)
    for j in range(-(-length // p)):
        if 0 <= table[j] < n:
            m = min(p, length - j * p)
            out[j * p:j * p + m] = pages[table[j], :, :m].transpose(1, 0, 2)
            there[j * p:j * p + m] = True
    return out, there


def attend(q, k, v, seen, scale):
    """One token ``[QH, D]`` over the rows ``seen``: zeros without any."""
    qh, d = q.shape
    out = np.zeros((qh, d))
    if not seen.any():
        return out
    group = qh // k.shape[1]
    for h in range(qh):
        s = (k[seen, h // group] @ q[h]) * scale
        e = np.exp(s - s.max())
        out[h] = (e / e.sum()) @ v[seen, h // group]
    return out


def decode_attention(q, keys, values, table, lengths, scale=None):
    b, qh, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros((b, qh, d))
    for i in range(b):
        (k, there), (v, _) = rows_of(keys, table[i], lengths[i]), rows_of(values, table[i], lengths[i])
        out[i] = attend(q[i], k, v, there, scale)
    return out.reshape(b, qh * d)


def prompt_attention(q, keys, values, table, lengths, starts, before, scale=None):
    """``before``: what the output held (padding keeps it)."""
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    out = before.copy().reshape(q.shape)
    for i in range(len(table)):
        (k, there), (v, _) = rows_of(keys, table[i], lengths[i]), rows_of(values, table[i], lengths[i])
        n = starts[i + 1] - starts[i]
        for t in range(n):
            seen = there & (np.arange(len(there)) <= len(there) - n + t)
            out[starts[i] + t] = attend(q[starts[i] + t], k, v, seen, scale)
    return out.reshape(before.shape)


def rope(x, position, weight, cos, sin, eps):
    """One head ``[D]``."""
    d = len(x)
    if weight is not None:
        x = x / math.sqrt((x * x).mean() + eps) * weight
    p = min(max(position, 0), len(cos) - 1)
    return x * cos[p] + np.concatenate((-x[d // 2:], x[:d // 2])) * sin[p]


def qk_rope(qkv, q_weight, k_weight, cos, sin, keys, values, table, lengths, starts, eps, before):
    """(q, keys, values) after the call; ``before``: what q held."""
    n, kh, p, d = keys.shape
    x = qkv.reshape(len(qkv), -1, d)
    qh = x.shape[1] - 2 * kh
    q, keys, values = before.copy(), keys.copy(), values.copy()
    for i in range(len(table)):
        count = starts[i + 1] - starts[i]
        for t in range(count):
            at, position = starts[i] + t, min(max(int(lengths[i]), 0), table.shape[1] * p) - count + t
            for h in range(qh):
                q[at, h] = rope(x[at, h], position, q_weight, cos, sin, eps)
            if position < 0 or position // p >= table.shape[1] or not 0 <= table[i, position // p] < n:
                continue
            page, row = table[i, position // p], position % p
            for h in range(kh):
                keys[page, h, row] = rope(x[at, qh + h], position, k_weight, cos, sin, eps)
                values[page, h, row] = x[at, qh + kh + h]
    return q, keys, values


def sample(logits, u, temperature, top_k, top_p, min_p):
    """(index, least distance of a decision to its border, in shares of the kept weight) of one row."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    if x.max() == -np.inf:
        return -1, math.inf
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return int(order[0]), math.inf
    with np.errstate(invalid="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / float(temperature)))
    order = order[:top_k] if 0 < top_k < len(x) else order
    ws, near = w[order], math.inf
    if top_p < 1:
        before = np.concatenate(([0.0], np.cumsum(ws)[:-1]))
        total = math.fsum(ws)
        keep = before <= float(top_p) * total
        near = np.abs(before[1:] / total - float(top_p)).min() if len(ws) > 1 else math.inf
        order, ws = order[keep], ws[keep]
    if min_p > 0:
        near = min(near, np.abs(ws - min(float(min_p), 1.0)).min()) if min_p < 1 else near
        order = order[ws >= min(float(min_p), 1.0)]
    kept = np.zeros(len(x))
    kept[order] = w[order]
    through = np.cumsum(kept)
    goal = float(u) * through[-1]
    near = min(near, np.abs(through - goal).min() / through[-1])
    drawn = int((through <= goal).sum())
    return (drawn if drawn < len(x) else int(np.nonzero(kept)[0][-1])), near
