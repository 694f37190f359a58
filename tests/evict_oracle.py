"""Plain float64 forms (CPU torch) of the paged cache's operators beyond causal
attention: draft trees with their statistics, attention weights by key, the
positions to keep and their move. Written from their definitions."""
import math

import torch

import paged_oracle as po

PAGE, D = po.PAGE, po.D


def tree_words(parents, words):
    """int64 words of each row: its ancestors' bits and its own."""
    bits, rows = [], []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    for x in bits:
        w = [x >> 64 * k & (1 << 64) - 1 for k in range(words)]
        rows.append([v - (1 << 64) if v >> 63 else v for v in w])
    return rows


def rows_of(c, b, max_q=None):
    """(first row, rows, position of the first, keys) of sequence b, cut as a call cuts."""
    q0, ql = c["qs"][b], c["qs"][b + 1] - c["qs"][b]
    p0 = max(c["kv_len"][b], 0) - ql
    ql = min(ql, c["max_q"] if max_q is None else max_q)
    return q0, ql, p0, max(p0 + ql, 0)


def attend(q, K, seen, V=None, gate=None):
    """One head's rows: q [n, D], K, V [kv, D], seen [n, kv]. (out, its bound, lse, its
    bound, x). The bounds are paged_oracle.attention's; lse's: fp32 scores (256 products,
    summed in any order), exp2 and log2 one step each, l a sum of kv terms in any order."""
    x = q @ K.T
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    m = x.amax(-1, keepdim=True)
    none = torch.isinf(m[:, 0])
    p = torch.where(seen, torch.exp2(x - torch.where(torch.isinf(m), 0.0, m)), 0.0)
    l = p.sum(-1, keepdim=True)
    lse = torch.where(none, -math.inf, (m + torch.log2(l))[:, 0])
    mag = torch.where(seen, q.abs() @ K.abs().T, 0.0).amax(-1)
    tol_lse = 2 * 256 * 2.0 ** -24 * mag + (2.0 ** -22 + K.shape[0] * 2.0 ** -24) / math.log(2.0) \
        + torch.where(none, 0.0, lse).abs() * 2.0 ** -23
    if V is None:
        return lse, tol_lse, x
    pr = p / torch.where(l > 0, l, 1.0)
    g = 1.0 if gate is None else torch.sigmoid(gate)
    eps = (2.0 ** -8 + 2 * math.log(2.0) * 256 * 2.0 ** -24 * mag + 2.0 ** -19)[:, None]
    o = pr @ V
    tol = (pr @ V.abs() * eps + o.abs() * 2.0 ** -8 * (1 + 2.0 ** -7)) * g + 1e-30
    return o * g, tol, lse, tol_lse


def weights(q, lse, K, seen):
    """One kv-head: q [n, G, D], lse [n, G], K [kv, D], seen [n, kv]: the sum over rows
    and heads of 2^(q.k - lse), and its bound: fp32 scores as above, their difference with
    lse rounded, exp2 two steps, the sum of n G terms in any order."""
    n, G = lse.shape
    w, tol = torch.zeros(K.shape[0], dtype=torch.float64), torch.zeros(K.shape[0], dtype=torch.float64)
    for g in range(G):
        x, mag = q[:, g] @ K.T, q[:, g].abs() @ K.abs().T
        at = torch.where(torch.isinf(lse[:, g]), 0.0, lse[:, g])[:, None]
        p = torch.where(seen & ~torch.isinf(lse[:, g])[:, None], torch.exp2(x - at), 0.0)
        w += p.sum(0)
        rel = math.log(2.0) * (2 * 256 * 2.0 ** -24 * mag + 2.0 ** -23 * (x.abs() + at.abs())) + 2.0 ** -21
        tol += (p * rel).sum(0)
    return w, tol + w * (n * G + 8) * 2.0 ** -24 + 1e-35


def order(w):
    """A key that sorts fp32 weights as the selection does: NaN first, -0 as 0."""
    return (0, 0.0) if math.isnan(w) else (1, -w + 0.0)


def select(w, kv, budget, sinks, recent):
    """Positions kept of weights w[0 .. kv - 1] (a missing page's: None)."""
    n = min(kv, budget)
    if kv <= budget:
        return list(range(kv))
    mid = sorted(range(sinks, kv - recent),
                 key=lambda j: ((2, 0.0) if w[j] is None else order(w[j]), j))
    return sorted(list(range(sinks)) + list(range(kv - recent, kv)) + mid[:n - sinks - recent])
