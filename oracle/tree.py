"""Tree-speculation operators restated in 64 bits, node by node (test infrastructure only)."""

from __future__ import annotations

import math
from typing import Optional

import numpy as np


def ancestors(parents: np.ndarray):
    """(words uint64 [B, T], depths [B, T]) by walking every node up to its root."""
    B, T = parents.shape
    bits, depth = np.zeros((B, T), np.uint64), np.zeros((B, T), np.int32)
    for b in range(B):
        for i in range(T):
            node, word, n = i, 0, 0
            while True:
                up = int(parents[b, node])
                if up != -1 and not 0 <= up < node:
                    word = n = 0  # belongs to no tree
                    break
                word |= 1 << node
                if up == -1:
                    break
                node, n = up, n + 1
            bits[b, i], depth[b, i] = word, n
    return bits, depth


def dequant(t, bits: int):
    """fp64 rows of an MLX tuple (numpy int32 words, fp64 scales, fp64 biases), or of a bf16 array given as fp64."""
    if not bits:
        return t
    w, s, b = t
    sh = np.arange(0, 32, bits, dtype=np.uint32)
    c = ((w.view(np.uint32)[..., None] >> sh) & (2 ** bits - 1)).reshape(*w.shape[:-1], -1).astype(np.float64)
    return c * np.repeat(s, 64, -1) + np.repeat(b, 64, -1)


def attention(q, k, v, length: int, words, T: int, scale: float):
    """One sequence: q fp64 [Hq, L, D], k/v fp64 [Hkv, rows, D] -> (out, sum p |v|) fp64 [Hq, L, D]."""
    Hq, L, D = q.shape
    G = Hq // k.shape[0]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(L):
        seen = list(range(min(length, k.shape[1])))
        seen += [length + j for j in range(T) if int(words[i]) >> j & 1 and length + j < k.shape[1]]
        if not seen:
            continue
        for h in range(Hq):
            s = scale * (k[h // G, seen] @ q[h, i])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h, i] = p @ v[h // G, seen]
            mag[h, i] = p @ np.abs(v[h // G, seen])
    return out, mag


def process_row(x, counts=None, penalties=None, path=(), bias=None, mask=None):
    """One row: x fp64 [V]; path = tokens on the node's own path; bias = [(id, value)]; mask = words."""
    y, V = x.copy(), len(x)
    c = np.zeros(V, np.int64) if counts is None else counts.astype(np.int64).copy()
    for t in path:
        if 0 <= t < V:
            c[t] += 1
    if penalties is not None:
        rep, pres, freq = (float(z) for z in penalties)
        for w in np.nonzero(c > 0)[0]:
            z = y[w] * rep if y[w] < 0 else y[w] / rep
            y[w] = z - pres - freq * c[w]
    for w, val in dict((int(i), float(z)) for i, z in (bias or [])).items():  # the last entry of a token counts
        if 0 <= w < V:
            y[w] += val
    if mask is not None:
        for w in range(V):
            if not (int(mask[w >> 5]) >> (w & 31)) & 1:
                y[w] = -math.inf
    return y


def choice(row) -> int:
    """First index of the largest value, NaN never; -1 where nothing is left."""
    best, at = -math.inf, -1
    for w, z in enumerate(row):
        if z > best:
            best, at = z, w
    return at


def accept(parents, tokens, picks):
    """One sequence: (path, next)."""
    path, cur = [0], 0
    while True:
        nxt: Optional[int] = None
        for i in range(cur + 1, len(parents)):
            if parents[i] == cur and tokens[i] == picks[cur]:
                nxt = i
                break
        if nxt is None:
            return path, int(picks[cur])
        path.append(nxt)
        cur = nxt
