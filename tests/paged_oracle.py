"""Plain float64 forms of the paged K/V cache's operators (CPU torch), written
from their definitions, and the inputs that the tests of both share."""
import math

import torch

PAGE, D = 64, 256
LOG2E = 1.4426950408889634


def e4m3_round(x):
    """float64 to the nearest e4m3 value, ties to even (|x| <= 448)."""
    a = x.abs()
    e = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a))))
    e = torch.where(torch.exp2(e) > a, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= a, e + 1, e)
    step = torch.exp2((e - 3).clamp(min=-9))
    return torch.round(x / step) * step


def row_scale(a):
    """2^e, e the least integer in [-100, 120] with a <= 448 * 2^e."""
    out = torch.empty_like(a)
    for i, v in enumerate(a.flatten().tolist()):
        e = -100
        while e < 120 and v > 448.0 * 2.0 ** e:
            e += 1
        out.view(-1)[i] = 2.0 ** e
    return out


def quantise(x, dim):
    """(e4m3 values, scales) of the rows of x along dim, in float64."""
    s = row_scale(x.abs().amax(dim))
    return e4m3_round(x / s.unsqueeze(dim)), s


def norm_rope(x, w, cos, sin, rot, eps):
    """Rows of x [..., D] in float64: RMSNorm, then rotate_half of the first rot dims."""
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    h = rot // 2
    a, b = y[..., :h], y[..., h:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], -1)


def slots(q_start, kv_len, page_table, b, num_pages):
    """[(row, position, page, slot)] of sequence b's new tokens that have a slot."""
    out, q0, q1 = [], q_start[b], q_start[b + 1]
    for n in range(q0, q1):
        p = kv_len[b] - (q1 - q0) + n - q0
        if p < 0 or p // PAGE >= len(page_table[b]):
            continue
        page = page_table[b][p // PAGE]
        if 0 <= page < num_pages:
            out.append((n, p, page, p % PAGE))
    return out


def attention(q, gate, K, V, keys, q_start, kv_len, window, sinks):
    """out [N, Hq, D] (NaN where no sequence has the row) and the bound on a
    kernel's error that rounds p to bf16 and the result to bf16: half a step
    each, the first weighted by sum p |v| / l, and fp32 scores (256 products
    summed in any order: 256 half steps of sum |q k|, twice, in ln 2 units of
    the exponent). K, V: per sequence [Hkv, kv, D]; keys: per sequence a bool
    [kv], whether the key is there at all."""
    N, Hq = q.shape[0], q.shape[1]
    out = torch.full((N, Hq, D), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(len(kv_len)):
        q0, q1, kv = q_start[b], q_start[b + 1], kv_len[b]
        j = torch.arange(kv)
        for n in range(q0, q1):
            p = kv - (q1 - q0) + n - q0
            seen = (j <= p) & keys[b]
            if window:
                seen &= (j > p - window) | (j < sinks)
            for h in range(Hq):
                kh = h // (Hq // K[b].shape[0])
                g = 1.0 if gate is None else torch.sigmoid(gate[n, h])
                if not seen.any():
                    out[n, h] = 0.0
                    continue
                k, v = K[b][kh][seen], V[b][kh][seen]
                x = k @ q[n, h]
                pr = torch.exp2(x - x.max())
                pr = pr / pr.sum()
                o = pr @ v
                mag = (k.abs() @ q[n, h].abs()).max()
                eps = 2.0 ** -8 + 2 * math.log(2.0) * 256 * 2.0 ** -24 * mag + 2.0 ** -19
                out[n, h] = o * g
                tol[n, h] = (pr @ v.abs() * eps + o.abs() * 2.0 ** -8 * (1 + 2.0 ** -7)) * g + 1e-30
    return out, tol
