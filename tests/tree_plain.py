"""Plain forms, in float64, of the operators of drafted tokens."""
import math
import random

import numpy as np
import torch


def random_tree(rng, rows, width):
    """Parents (-1 of row 0), each before its children."""
    return [-1] + [i - 1 if rng.random() < 0.4 else rng.randrange(max(0, i - 2 * width), i) for i in range(1, rows)]


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def ancestors(parents):
    """Truth values [rows, rows]: row i sees row j."""
    see = np.zeros((len(parents), len(parents)), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


def words(see, width):
    """Truth values [rows, rows] as int32 [rows, width], 32 a word."""
    out = np.zeros((see.shape[0], width), dtype=np.uint32)
    for j in range(see.shape[1]):
        out[:, j // 32] |= see[:, j].astype(np.uint32) << np.uint32(j % 32)
    return out.view(np.int32)


def attention(q, k, v, start, positions, see, scale, window):
    """One request: q [rows, nh, hd], k and v [start + rows, nkv, hd], see [rows, rows]. Returns (out, sum of weights times |v|, largest sum of |q||k| scale)."""
    q, k, v = q.double(), k.double(), v.double()
    rows, nh, hd = q.shape
    nkv = k.shape[1]
    seen = torch.zeros(rows, start + rows, dtype=torch.bool)
    for i in range(rows):
        p = int(positions[i])
        for j in range(start):
            seen[i, j] = not window or p - j < window
        for j in range(rows):
            seen[i, start + j] = bool(see[i, j]) and (not window or p - int(positions[j]) < window)
    seen = seen.to(q.device)
    out, size, reach = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for h in range(nh):
        kh, vh = k[:, h * nkv // nh], v[:, h * nkv // nh]
        s = (q[:, h] @ kh.T * scale)
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(-1, keepdim=True)
        w = torch.where(seen, torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top)), torch.zeros_like(s))
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, w)
        # (what is masked is no part of a sum, whatever it holds)
        for i in range(rows):
            at = seen[i].nonzero()[:, 0]
            out[i, h] = w[i, at] @ vh[at]
            size[i, h] = w[i, at] @ vh[at].abs()
            if len(at):
                reach = max(reach, float((q[i, h].abs() @ kh[at].abs().T).max()) * abs(scale))
    return out, size, reach


def tolerance(out, size, reach, hd, keys, dtype):
    """How far a kernel may be from ``attention``: scores are sums of hd products in float32, one exponential of each (ex2.approx: 2^-22), sums of ``keys``
    weights; in bfloat16 weights and the result are rounded, half a step (2^-8) of each."""
    delta = (hd + 4) * 2.0 ** -24 * reach * 1.5 + 2.0 ** -21
    tol = size * (2 * delta + (keys + 8) * 2.0 ** -24)
    return tol + 2.0 ** -8 * (size + out.abs()) if dtype == torch.bfloat16 else tol + 2.0 ** -24 * out.abs()


def softmax(x, t):
    x = np.asarray(x, dtype=np.float64)
    e = np.exp((x - x.max()) / float(np.float32(t)))
    return e / e.sum()


def draw(weights, u):
    upto = np.cumsum(weights)
    return int(min(np.searchsorted(upto, float(u) * upto[-1], side="right"), len(weights) - 1))


def verify(logits, tokens, parents, uniform, temperature, draft=None):
    """One request, by walking: (kept rows, token that follows)."""
    cur, kept = 0, [0]
    while True:
        x = logits[cur].astype(np.float64)
        children = [c for c in range(cur + 1, len(parents)) if parents[c] == cur]
        if not temperature > 0:
            token = -1 if np.isnan(x).all() else int(np.nanargmax(x))
            go = next((c for c in children if tokens[c] == token and token >= 0), None)
        else:
            rows = [x] + ([draft[cur].astype(np.float64)] if draft is not None else [])
            if any(np.isnan(r).any() or (r == np.inf).any() or (r == -np.inf).all() for r in rows):
                return kept, -1
            r = softmax(x, temperature)
            if draft is None:
                token = draw(r, uniform[cur, 1])
                go = next((c for c in children if tokens[c] == token), None)
            else:
                q, p, go = softmax(rows[1], temperature), r, None
                for c in children:
                    t = int(tokens[c])
                    if not 0 <= t < len(x):
                        continue
                    if float(uniform[c, 0]) * q[t] * r.sum() < r[t]:
                        go = c
                        break
                    r = np.maximum(r - r.sum() * q, 0)
                    if not r.sum() > 0:
                        r = p
                        break
                token = None if go is not None else draw(r, uniform[cur, 1])
        if go is None:
            return kept, token
        cur = go
        kept.append(go)
