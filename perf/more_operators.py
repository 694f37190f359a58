"""More operators of the paged K/V cache as cases that can be timed and compared:
writing tokens whose rotary positions have several axes, attention of a tree of
drafted tokens with its softmax statistics, and eviction: attention weights
accumulated by key, the positions to keep, and their move to the front.

A page holds 64 tokens of every kv-head, K as [64][256] and V transposed as
[256][64], in bf16 or in e4m3 with one power-of-two scale per token and kv-head.
Sequence b's new tokens are rows q_start[b] .. q_start[b + 1] of the call and its
last keys: token i of ql has position kv_len[b] - ql + i.

Kinds of case
  prep     norm + RoPE of q and K, and K / V written into the pages; frequency i
           turns by the position on axis i's axis (time, height or width)
  tree     attention of drafted tokens over their sequences' pages: a token sees
           the committed keys and, of the drafted ones, its ancestors and itself;
           with lse, the base-2 log of the softmax's sum, for each row and head
  weights  prev + the sum over rows and heads of 2^(q.k - lse), for each key
  select   the positions of a budget's keys: the first `sinks`, the last
           `recent`, the heaviest of the others (ties: the lowest), ascending
  keep     K, V, scales and weights of a list of positions moved to the front: an
           evicted cache into other pages, or a draft's accepted path in place

Listed head counts are those of the repository's presets and tests (16/4 and
8/2 heads of 256); drawn ones have other group sizes too. Lengths go from one
token to 16384 keys.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

D = 256            # head dim
PAGE = 64          # tokens a page
ROT = 64           # rotary dims
THETA = 1e7
EPS = 1e-6
Q_SCALE = 1.4426950408889634 / 16  # head_dim^-1/2 log2 e
E4M3_MAX = 448.0


# ---- the cases ---------------------------------------------------------------
def listed():
    h = dict(Hq=16, Hkv=4)
    return [
        # one decoding step of 64 sequences after pictures: a token each
        dict(name="prep_64x1_e4m3", kind="prep", B=64, q=1, kv=1000, even=False, e4m3=True,
             sections="11,11,10", mixed=True, **h),
        # two prompts, pictures of many patches amid text
        dict(name="prep_2x2500_bf16", kind="prep", B=2, q=2500, kv=2500, even=True, e4m3=False,
             sections="11,11,10", mixed=True, **h),
        # the latency of one draft tree on a short context
        dict(name="tree_1x26_on_530_bf16", kind="tree", B=1, q=26, kv=530, even=True, e4m3=False,
             **h),
        # a verification step of 64 sequences of up to 4096 keys in 8 bits
        dict(name="tree_64x16_on_4096_e4m3", kind="tree", B=64, q=16, kv=4096, even=False,
             e4m3=True, **h),
        # large trees on long documents
        dict(name="tree_8x64_on_8192_bf16", kind="tree", B=8, q=64, kv=8192, even=False,
             e4m3=False, **h),
        # a decoding step's weights, 64 sequences of up to 4096 keys in 8 bits
        dict(name="weights_64x1_on_4096_e4m3", kind="weights", B=64, q=1, kv=4096, even=False,
             e4m3=True, **h),
        # a prompt's last 32 tokens observing it, 16 sequences
        dict(name="weights_16x32_on_2048_bf16", kind="weights", B=16, q=32, kv=2048, even=False,
             e4m3=False, **h),
        # the second half of a document of 8192
        dict(name="weights_4096_on_8192_bf16", kind="weights", B=1, q=4096, kv=8192, even=True,
             e4m3=False, **h),
        # one long context to a quarter
        dict(name="select_1x8192_to_2048", kind="select", B=1, kv=8192, even=True, budget=2048,
             sinks=4, recent=256, **h),
        # 64 sequences of up to 4096 keys to 1024 each
        dict(name="select_64x4096_to_1024", kind="select", B=64, kv=4096, even=False, budget=1024,
             sinks=4, recent=64, **h),
        # evicted caches of 16 sequences into other pages
        dict(name="keep_16x4096_to_1024_bf16", kind="keep", B=16, kv=4096, even=False, n=1024,
             e4m3=False, inplace=False, **h),
        # the accepted paths of 64 draft trees in place
        dict(name="keep_64x6_of_32_e4m3", kind="keep", B=64, kv=4096, even=False, n=6, tree=32,
             e4m3=True, inplace=True, **h),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prep", "tree", "tree", "tree", "weights", "weights", "weights", "select",
                       "keep"])
    Hq, Hkv = rng.choice([(16, 4), (16, 4), (8, 2), (4, 1), (16, 2), (6, 1), (4, 4)])
    c = dict(kind=kind, Hq=Hq, Hkv=Hkv, even=False, e4m3=rng.random() < 0.5)
    if kind == "prep":
        c["q"] = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        c["B"] = _log_int(rng, 1, max(1, min(64, 5000 // c["q"])))
        c["kv"] = c["q"] + _log_int(rng, 1, 1000)
        c["sections"] = rng.choice(["11,11,10", "11,11,10", "16,8,8", "12,10,6,4", "16,16"])
        c["mixed"] = rng.random() < 0.5
    elif kind == "tree":
        c["q"] = rng.choice([1, _log_int(rng, 2, 64), _log_int(rng, 2, 64), _log_int(rng, 65, 256)])
        c["kv"] = c["q"] + _log_int(rng, 1, 8192)
        c["B"] = _log_int(rng, 1, max(1, min(64, 8 * 64 * 8192 // (c["q"] * c["kv"]),
                                             64 * 4096 // c["kv"])))
    elif kind == "weights":
        c["q"] = 1 if rng.random() < 0.3 else _log_int(rng, 2, 4096)
        c["kv"] = c["q"] + _log_int(rng, 1, max(2, 8192 - c["q"]))
        c["B"] = _log_int(rng, 1, max(1, min(64, 4096 * 6000 // (c["q"] * c["kv"]),
                                             64 * 4096 // c["kv"])))
    elif kind == "select":
        c.pop("e4m3")
        c["kv"] = _log_int(rng, 1, 16384)
        c["B"] = _log_int(rng, 1, max(1, min(64, 64 * 4096 // c["kv"])))
        c["budget"] = _log_int(rng, 1, c["kv"])
        c["sinks"] = rng.choice([0, min(4, c["budget"])])
        c["recent"] = rng.randint(0, c["budget"] - c["sinks"])
    else:
        c["inplace"] = rng.random() < 0.5
        c["kv"] = _log_int(rng, 64, 8192)
        if c["inplace"]:
            c["tree"] = rng.randint(2, 64)
            c["n"] = rng.randint(1, max(1, min(8, c["tree"] // 2)))
        else:
            c["n"] = _log_int(rng, 1, c["kv"])
        c["B"] = _log_int(rng, 1, max(1, min(64, 16 * 4096 // c["kv"])))
    return c


def _lens(case):
    """(new tokens, keys) of each sequence: q and kv at most, the first one's in
    full; unevenly the others from 1 and from kv / 4 (the sizes alone decide)."""
    B, kv, q = case["B"], case["kv"], case.get("q", 0)
    r = random.Random(B * 1000003 + kv * 1009 + q)
    out = []
    for b in range(B):
        n = q if case["even"] or b == 0 else r.randint(1, q) if q else 0
        k = kv if case["even"] or b == 0 else r.randint(max(1, kv // 4), kv)
        out.append((n, max(n, k, case.get("tree", 0))))
    return out


def _kept(case):
    """What each sequence keeps: at most n, and no more than it has."""
    return [min(case["n"], k) for _, k in _lens(case)]


# ---- inputs -------------------------------------------------------------------
def _rope_table(npos):
    """(cos, sin) of the fp32 angle fl(theta^(-2i/rot)) p, as the engine builds it."""
    inv = torch.tensor([THETA ** (-2.0 * i / ROT) for i in range(ROT // 2)], device="cuda",
                       dtype=torch.float64).float()
    a = (inv * torch.arange(npos, device="cuda").float()[:, None]).double()
    return torch.stack([a.cos(), a.sin()], dim=-1).float().contiguous()


def _quantise(x, dim):
    """(e4m3, scale): the power of two 2^e, e the least integer with max |x| <= 448 2^e."""
    m, e = torch.frexp(x.abs().amax(dim=dim, keepdim=True))
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-100, 120)
    two_to = lambda n: ((n + 127) << 23).view(torch.float32)
    return (x * two_to(-e)).to(torch.float8_e4m3fn), two_to(e).squeeze(dim)


def _positions(r, n, axes, mixed):
    """Positions of n tokens on each axis: text (the same on all) and, mixed in,
    pictures, whose patches share a time and differ in height and width."""
    out, at = [[] for _ in range(axes)], r.randint(0, 500)
    while len(out[0]) < n:
        if mixed and r.random() < 0.3:
            h, w = r.randint(2, 24), r.randint(2, 24)
            for y in range(h):
                for x in range(w):
                    for a in range(axes):
                        out[a].append(at + (0 if a == 0 else y if a % 2 == 1 else x))
            at += max(h, w)
        else:
            for _ in range(r.randint(1, 200)):
                for a in range(axes):
                    out[a].append(at)
                at += 1
    return [o[-n:] for o in out]


def _axis_of(case):
    """The axis of each of the ROT / 2 frequencies: in turn while their sections last,
    the rest time's (three axes), or one section after the other."""
    sec = [int(x) for x in case["sections"].split(",")]
    if case["sections"] == "11,11,10":
        return [i % 3 if i % 3 and i < 3 * sec[i % 3] else 0 for i in range(ROT // 2)]
    return [a for a, n in enumerate(sec) for _ in range(n)]


def _draft(r, n):
    """Parents of n drafted tokens, each before its children; -1: the last committed."""
    return [-1 if i == 0 or r.random() < 0.1 else r.randrange(max(0, i - 20), i)
            for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    r = random.Random(int(seed))
    Hq, Hkv, B, e4m3 = case["Hq"], case["Hkv"], case["B"], case.get("e4m3", False)
    kind, lens = case["kind"], _lens(case)
    N, max_q, max_kv = sum(n for n, _ in lens), max(n for n, _ in lens), max(k for _, k in lens)
    need = [-(-k // PAGE) for _, k in lens]
    max_pages = max(need)
    keep_pages = [-(-n // PAGE) for n in _kept(case)] if kind == "keep" else [0]
    num_pages = sum(need) + sum(keep_pages) + 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    s = dict(case=case, N=N, max_q=max_q, max_kv=max_kv, kv_len=i32([k for _, k in lens]))
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s["q_start"] = i32(starts)
    # the sequences' pages lie anywhere in the pool
    perm = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    at = 0

    def table(counts):
        nonlocal at
        t = torch.zeros(B, max(counts), dtype=torch.int32, device="cuda")
        for b, n in enumerate(counts):
            t[b, :n] = perm[at:at + n]
            at += n
        return t

    s["page_table"] = table(need)
    randn = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
    if kind in ("weights", "select", "keep"):
        # a few keys have most of the weight, some none
        w = torch.exp(2 * randn(num_pages, Hkv, PAGE))
        s["weights"] = torch.where(w < 0.1, 0.0, w)
    if kind == "select":
        s["keep"] = torch.full((B, Hkv, case["budget"]), -1, dtype=torch.int32, device="cuda")
        s["keep_len"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        return s
    # the pool: every slot holds something, as after use by other sequences
    k, vt = randn(num_pages, Hkv, PAGE, D), randn(num_pages, Hkv, D, PAGE)
    if e4m3:
        s["k"], s["k_scale"] = _quantise(k, 3)
        s["vt"], s["v_scale"] = _quantise(vt, 2)
    else:
        s["k"], s["vt"], s["k_scale"], s["v_scale"] = k.bfloat16(), vt.bfloat16(), None, None
    del k, vt
    if kind == "keep":
        kept = _kept(case)
        s["keep_len"] = i32(kept)
        if case["inplace"]:
            # the paths lie behind the slots that they go to (first levels are wider
            # than the paths are long), so that a pass leaves its own input
            T = case["tree"]
            s["dst"] = i32([kv - T for _, kv in lens])
            s["keep"] = i32([[[kv - T + x for x in sorted(r.sample(range(n, T), n))]
                              + [0] * (case["n"] - n)] for n, (_, kv) in zip(kept, lens)])
            s["to"] = None
        else:
            s["dst"] = None
            # each head's own positions
            live = torch.arange(max_kv, device="cuda") < s["kv_len"][:, None]
            x = torch.rand(B, Hkv, max_kv, device="cuda", generator=g)
            x = torch.where(live[:, None], x, 2.0).argsort(-1)[..., :case["n"]]
            first = torch.arange(case["n"], device="cuda") < s["keep_len"][:, None]
            x = torch.where(first[:, None], x, max_kv).sort(-1).values
            s["keep"] = torch.where(first[:, None], x, 0).int().contiguous()
            s["to"] = table(keep_pages)
        return s
    if kind == "prep":
        axis_of = _axis_of(case)
        A = max(axis_of) + 1
        pos = [[] for _ in range(A)]
        for n, _ in lens:
            for a, p in enumerate(_positions(r, n, A, case["mixed"])):
                pos[a] += p
        s["pos"], s["axis_of"] = i32(pos), axis_of
        s["rope"] = _rope_table(max(map(max, pos)) + 1)
        s["proj"] = randn(N, Hq * 2 * D + 2 * Hkv * D).bfloat16()
        s["q_w"], s["k_w"] = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
        s["q_out"] = torch.empty(N, Hq, D, dtype=torch.bfloat16, device="cuda")
        return s
    s["q"] = (randn(N, Hq, D) * Q_SCALE).bfloat16()
    if kind == "weights":
        s["prev"], s["weights"] = s["weights"], torch.zeros_like(s["weights"])
        # the statistics that the attention of the same rows gives
        s["lse"] = torch.zeros(N, Hq, device="cuda")
        for b, (n, kv) in enumerate(lens):
            kk, q0 = _one_k(s, b, kv), starts[b]
            hidden = _behind(kv - n, n, kv)
            for h in range(Hq):
                x = s["q"][q0:q0 + n, h].float() @ kk[h // (Hq // Hkv)].t()
                x.masked_fill_(hidden, -math.inf)
                s["lse"][q0:q0 + n, h] = torch.logsumexp(x * math.log(2.0), -1) / math.log(2.0)
        return s
    # the gates lie in the layer's projection rows [q | gate per q-head][K][V]
    s["proj"] = randn(N, Hq * 2 * D + 2 * Hkv * D).bfloat16()
    s["parents"], s["words"] = [], -(-max_q // 64)
    rows = []
    for n, _ in lens:
        parents, bits = _draft(r, n), []
        for i, p in enumerate(parents):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        s["parents"].append(parents)
        rows += [[x >> 64 * w & (1 << 64) - 1 for w in range(s["words"])] for x in bits]
    s["tree"] = torch.from_numpy(np.array(rows, dtype=np.uint64).view(np.int64)).cuda()
    s["out"] = torch.empty(N, Hq * D, dtype=torch.bfloat16, device="cuda")
    s["lse"] = torch.empty(N, Hq, device="cuda")
    return s


def _behind(p0, n, kv):
    """Which of the keys 0 .. kv - 1 the rows at positions p0 .. p0 + n - 1 do not see."""
    p = torch.arange(p0, p0 + n, device="cuda")
    return torch.arange(kv, device="cuda") > p[:, None]


def _one_k(s, b, kv):
    """K [Hkv, kv, D] of sequence b, in 32 bits."""
    at = s["page_table"][b, :-(-kv // PAGE)].long()
    if s["case"]["e4m3"]:
        k = s["k"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
        k = k * s["k_scale"][at][..., None]
    else:
        k = s["k"][at].float()
    return k.transpose(0, 1).flatten(1, 2)[:, :kv]


# ---- one pass -------------------------------------------------------------------
def _ops():
    pkg = os.path.join(_ROOT, "cu-jev_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from cujev import ops
    return ops


def run(s):
    if own:
        return _OWN[s["case"]["kind"]](_ops(), s, s["case"])
    return _PLAIN[s["case"]["kind"]](s)


def _pages(ops, s):
    if "pages" not in s:  # a user's program keeps its pool
        s["pages"] = ops.KvPages(s["k"], s["vt"], s["k_scale"], s["v_scale"])
    return s["pages"]


def _own_prep(ops, s, c):
    if "axes" not in s:  # a model's, made once
        s["axes"] = ops.RopeAxes(s["axis_of"])
    ops.attn_prep_paged(s["proj"], s["q_w"], s["k_w"], s["pos"], s["q_start"], s["kv_len"],
                        s["page_table"], c["Hq"], ROT, s["rope"], EPS, Q_SCALE, s["q_out"],
                        _pages(ops, s), axes=s["axes"])
    return _pool(s, s["q_out"])


def _own_tree(ops, s, c):
    if "ws" not in s:  # a user's program keeps one for its largest call
        n = ops.attention_paged_ws_bytes(s["N"], c["B"], s["max_q"], s["max_kv"], c["Hq"],
                                         c["Hkv"], e4m3=c["e4m3"])
        s["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
    ops.attention_paged(s["q"], s["proj"][:, D:], s["proj"].stride(0), 2 * D, _pages(ops, s),
                        s["page_table"], s["q_start"], s["kv_len"], s["max_q"], s["max_kv"],
                        s["out"], ws=s["ws"], tree=s["tree"], lse=s["lse"])
    return s["out"], s["lse"]


def _own_weights(ops, s, c):
    ops.kv_weights(s["q"], s["lse"], _pages(ops, s), s["page_table"], s["q_start"], s["kv_len"],
                   s["max_q"], s["max_kv"], s["weights"], prev=s["prev"])
    return s["weights"]


def _own_select(ops, s, c):
    ops.kv_select(s["weights"], s["page_table"], s["kv_len"], s["max_kv"], c["budget"], s["keep"],
                  s["keep_len"], sinks=c["sinks"], recent=c["recent"])
    return s["keep"], s["keep_len"]


def _own_keep(ops, s, c):
    ops.kv_keep(_pages(ops, s), s["page_table"], s["keep"], s["keep_len"], dst=s["dst"],
                to_table=s["to"], weights=s["weights"])
    return _pool(s, s["weights"])


_OWN = dict(prep=_own_prep, tree=_own_tree, weights=_own_weights, select=_own_select,
            keep=_own_keep)


def _pool(s, other):
    """`other` and the pool as the pass leaves it (e4m3 values with their scales)."""
    return [other, s["k"], s["vt"]] + ([s["k_scale"], s["v_scale"]] if s["case"]["e4m3"] else [])


def _new_tokens(s):
    """(page, slot) of each new token."""
    ql = (s["q_start"][1:] - s["q_start"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(ql.numel(), device="cuda"), ql,
                                  output_size=s["N"])
    p = s["kv_len"].long()[seq] - s["q_start"].long()[1:][seq] + torch.arange(s["N"],
                                                                             device="cuda")
    return s["page_table"].long()[seq, p // PAGE], p % PAGE


def _norm_rope(x, w, cs):
    """RMSNorm of the rows of x [N, heads, D], then RoPE of the first ROT dims."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    a, b = x[..., :ROT // 2], x[..., ROT // 2:ROT]
    return torch.cat([a * c - b * sn, b * c + a * sn, x[..., ROT:]], dim=-1)


def _plain_prep(s):
    c, N = s["case"], s["N"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    axis = torch.tensor(s["axis_of"], device="cuda")
    # [N, ROT / 2]: the position that each frequency turns by
    p = s["pos"].long()[axis].t()
    cs = s["rope"][p, torch.arange(ROT // 2, device="cuda")]
    q = s["proj"][:, :Hq * 2 * D].reshape(N, Hq, 2 * D)[..., :D].float()
    k, v = s["proj"][:, Hq * 2 * D:].reshape(N, 2, Hkv, D).float().unbind(1)
    s["q_out"].copy_(_norm_rope(q, s["q_w"], cs) * Q_SCALE)
    k = _norm_rope(k, s["k_w"], cs)
    page, slot = _new_tokens(s)
    if c["e4m3"]:
        k, s["k_scale"][page, :, slot] = _quantise(k, 2)
        v, s["v_scale"][page, :, slot] = _quantise(v, 2)
        # elements of 8-bit floats move as bytes
        s["k"].view(torch.uint8)[page, :, slot] = k.view(torch.uint8)
        s["vt"].view(torch.uint8)[page, :, :, slot] = v.view(torch.uint8)
    else:
        s["k"][page, :, slot] = k.bfloat16()
        s["vt"][page, :, :, slot] = v.bfloat16()
    return _pool(s, s["q_out"])


def _gather(s, values=True):
    """K [B, Hkv, keys, D] and V [B, Hkv, keys, D] of the sequences' pages (keys
    padded to whole pages)."""
    pt = s["page_table"].long()
    if s["case"]["e4m3"]:  # an 8-bit float's elements are gathered as bytes
        k = s["k"].view(torch.uint8)[pt].view(torch.float8_e4m3fn).float()
        k = k * s["k_scale"][pt][..., None]
    else:
        k = s["k"][pt].float()
    B, Hkv = pt.shape[0], k.shape[2]
    k = k.transpose(1, 2).reshape(B, Hkv, -1, D)
    if not values:
        return k
    if s["case"]["e4m3"]:
        vt = s["vt"].view(torch.uint8)[pt].view(torch.float8_e4m3fn).float()
        vt = vt * s["v_scale"][pt][..., None, :]
    else:
        vt = s["vt"][pt].float()
    return k, vt.permute(0, 2, 1, 4, 3).reshape(B, Hkv, -1, D)


def _padded(s):
    """The rows of each sequence, padded to the longest one's: their numbers in the
    call [B, max_q], which of them are rows, their positions, and q [B, Hkv, G max_q, D]."""
    c, B, mq = s["case"], s["case"]["B"], s["max_q"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    G = Hq // Hkv
    q0, ql = s["q_start"].long()[:-1], (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(mq, device="cuda")
    there = i < ql[:, None]
    rows = torch.where(there, q0[:, None] + i, 0)
    p = s["kv_len"].long()[:, None] - ql[:, None] + i
    q = s["q"].float()[rows].reshape(B, mq, Hkv, G, D).permute(0, 2, 3, 1, 4)
    return rows, there, p, q.reshape(B, Hkv, G * mq, D)


def _plain_tree(s):
    c, B, mq = s["case"], s["case"]["B"], s["max_q"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    G = Hq // Hkv
    k, v = _gather(s)
    rows, there, p, q = _padded(s)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(B, Hkv, G, mq, -1)
    # key j is drafted token j - p0; before p0 all see it
    t = torch.arange(x.shape[-1], device="cuda") - p[:, :1]
    word = (t >> 6).clamp(0, s["words"] - 1)[:, None].expand(-1, mq, -1)
    bits = s["tree"][rows].gather(2, word) >> (t & 63)[:, None]
    seen = (t < 0)[:, None] | ((t < there.sum(1)[:, None])[:, None] & (bits & 1 != 0))
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp2(x - m)
    l = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, Hkv, G * mq, -1), v).reshape(B, Hkv, G, mq, D) / l
    o = o.permute(0, 3, 1, 2, 4).reshape(B, mq, Hq, D)[there]
    lse = (m + torch.log2(l)).squeeze(-1).permute(0, 3, 1, 2).reshape(B, mq, Hq)[there]
    gate = s["proj"][:, :Hq * 2 * D].reshape(-1, Hq, 2 * D)[..., D:].float()
    s["out"].copy_((o * torch.sigmoid(gate)).reshape(-1, Hq * D))
    s["lse"].copy_(lse)
    return s["out"], s["lse"]


def _plain_weights(s):
    c, B, mq = s["case"], s["case"]["B"], s["max_q"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    G = Hq // Hkv
    k = _gather(s, values=False)
    rows, there, p, q = _padded(s)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(B, Hkv, G, mq, -1)
    lse = s["lse"][rows].reshape(B, mq, Hkv, G).permute(0, 2, 3, 1)
    j = torch.arange(x.shape[-1], device="cuda")
    seen = there[..., None] & (j <= p[..., None])
    x = torch.exp2(x - lse[..., None])
    w = x.masked_fill_(~seen[:, None, None], 0.0).sum((2, 3))
    # prev counts for the keys before the new tokens
    pt = s["page_table"].long()
    prev = s["prev"][pt].transpose(1, 2).reshape(B, Hkv, -1)
    w += torch.where((j < p[:, :1])[:, None], prev, 0.0)
    live = (j < s["kv_len"][:, None])
    page, slot = pt.repeat_interleave(PAGE, 1)[live], (j % PAGE).expand(B, -1)[live]
    s["weights"][page, :, slot] = w.transpose(1, 2)[live]
    return s["weights"]


def _plain_select(s):
    c, B, Hkv = s["case"], s["case"]["B"], s["case"]["Hkv"]
    pt, kv, n = s["page_table"].long(), s["kv_len"].long()[:, None], c["budget"]
    w = s["weights"][pt].transpose(1, 2).reshape(B, Hkv, -1)
    j = torch.arange(w.shape[-1], device="cuda")
    safe = (j < kv) & ((j < c["sinks"]) | (j >= kv - c["recent"]))
    w = torch.where(safe[:, None], math.inf, torch.where((j < kv)[:, None], w, -math.inf))
    first = torch.argsort(w, dim=-1, descending=True, stable=True)[..., :n]
    first = torch.where(first < kv[..., None], first, w.shape[-1]).sort(-1).values
    m = first.shape[-1]
    count = kv.clamp(max=n)
    s["keep"][..., :m] = torch.where((j[:m] < count)[:, None], first.int(), s["keep"][..., :m])
    s["keep_len"].copy_(count[:, 0])
    return s["keep"], s["keep_len"]


def _plain_keep(s):
    c, B = s["case"], s["case"]["B"]
    heads = torch.arange(c["Hkv"], device="cuda")
    i = torch.arange(s["keep"].shape[-1], device="cuda")
    live = (i < s["keep_len"][:, None]).nonzero()
    b, i = live[:, :1], live[:, 1]
    src = s["keep"].long().expand(-1, c["Hkv"], -1)[b[:, 0], :, i]  # [moves, Hkv]
    dst = i[:, None] + (s["dst"].long()[b] if s["dst"] is not None else 0)
    to = s["page_table"] if s["to"] is None else s["to"]
    ps, pd = s["page_table"].long()[b, src // PAGE], to.long()[b, dst // PAGE]
    ss, sd = src % PAGE, dst % PAGE
    as_bytes = (lambda x: x.view(torch.uint8)) if c["e4m3"] else lambda x: x
    k, vt, w = as_bytes(s["k"]), as_bytes(s["vt"]), s["weights"]
    k[pd, heads, sd] = k[ps, heads, ss]
    vt[pd, heads, :, sd] = vt[ps, heads, :, ss]
    w[pd, heads, sd] = w[ps, heads, ss]
    if c["e4m3"]:
        for x in (s["k_scale"], s["v_scale"]):
            x[pd, heads, sd] = x[ps, heads, ss]
    return _pool(s, w)


_PLAIN = dict(prep=_plain_prep, tree=_plain_tree, weights=_plain_weights, select=_plain_select,
              keep=_plain_keep)


# ---- what a pass cannot do without ------------------------------------------------
def work(case):
    Hq, Hkv, kind = case["Hq"], case["Hkv"], case["kind"]
    lens, e4m3 = _lens(case), case.get("e4m3", False)
    N, keys = sum(n for n, _ in lens), sum(k for _, k in lens)
    half = Hkv * (D * (1 if e4m3 else 2) + (4 if e4m3 else 0))  # K or V of a cached token
    if kind == "prep":
        A = len(case["sections"].split(","))
        return dict(bytes=N * (Hq * D * 4 + Hkv * D * 4 + 2 * half + ROT * 4 + 4 * A),
                    flops=N * (Hq + Hkv) * D * 6)
    if kind == "select":
        return dict(bytes=4 * Hkv * (keys + sum(min(k, case["budget"]) for _, k in lens)),
                    flops=0)
    if kind == "keep":
        n = sum(_kept(case))
        return dict(bytes=n * (2 * (2 * half + 4 * Hkv) + (4 if case["inplace"] else 4 * Hkv)),
                    flops=0)
    if kind == "tree":  # a drafted token sees itself at least
        pairs = sum(n * (k - n + 1) for n, k in lens)
        return dict(bytes=keys * 2 * half + N * (Hq * (D * 6 + 4) + 8 * -(-case["q"] // 64)),
                    flops=4 * D * Hq * pairs)
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in lens)
    return dict(bytes=keys * (half + 4 * Hkv) + sum(k - n for n, k in lens) * 4 * Hkv
                + N * Hq * (D * 2 + 4), flops=2 * D * Hq * pairs)


# ---- the operators' definitions in 64 bits ------------------------------------------
def _to_e4m3(x):
    """x (float64, |x| <= 448) rounded to e4m3's values: 4 significant bits, ties to
    even, steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    return dict(prep=_exact_prep, tree=_exact_tree, weights=_exact_weights, select=_exact_select,
                keep=_exact_keep)[case["kind"]](s)


def _exact_scale(a):
    """2^ceil(log2(a / 448)) by comparison, within 2^-100 .. 2^120."""
    e = torch.ceil(torch.log2(a / E4M3_MAX).clamp(-100, 120))
    for d in (-1, 1):  # log2 may be a hair off next to a power of two
        up = a > E4M3_MAX * torch.exp2(e)
        down = a <= E4M3_MAX * torch.exp2(e - 1)
        e = torch.where(up, e + 1, torch.where(down, e - 1, e))
    return torch.exp2(e.clamp(-100, 120))


def _exact_prep(s):
    c = s["case"]
    Hq, Hkv, N = c["Hq"], c["Hkv"], s["N"]
    x = s["proj"].double()
    z = []
    for i, a in enumerate(s["axis_of"]):
        t = s["rope"][:, i].double()[s["pos"][a].long()]
        z.append(torch.complex(t[:, 0], t[:, 1]))
    z = torch.stack(z, 1)

    def rows(at, heads, step, w):
        y = torch.stack([x[:, at + h * step: at + h * step + D] for h in range(heads)], 1)
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS) * w.double()
        turned = torch.complex(y[..., :ROT // 2], y[..., ROT // 2:ROT]) * z[:, None]
        return torch.cat([turned.real, turned.imag, y[..., ROT:]], -1)

    q = rows(0, Hq, 2 * D, s["q_w"]) * Q_SCALE
    k = rows(Hq * 2 * D, Hkv, D, s["k_w"])
    v = x[:, Hq * 2 * D + Hkv * D:].reshape(N, Hkv, D)
    kp, vp = s["k"].double(), s["vt"].double()
    if c["e4m3"]:
        ks, vs = s["k_scale"].double(), s["v_scale"].double()
        sk, sv = _exact_scale(k.abs().amax(-1)), _exact_scale(v.abs().amax(-1))
        k, v = _to_e4m3(k / sk[..., None]), _to_e4m3(v / sv[..., None])
    page, slot = [], []
    table = s["page_table"].tolist()
    for b, (ql, kv) in enumerate(_lens(c)):
        for p in range(kv - ql, kv):
            page.append(table[b][p // PAGE])
            slot.append(p % PAGE)
    page, slot = torch.tensor(page, device="cuda"), torch.tensor(slot, device="cuda")
    kp[page, :, slot], vp[page, :, :, slot] = k, v
    if not c["e4m3"]:
        return [q, kp, vp]
    ks[page, :, slot], vs[page, :, slot] = sk, sv
    return [q, kp, vp, ks, vs]


def _exact_cache(s, b, kv):
    """K and V [Hkv, kv, D] of sequence b in float64."""
    at = s["page_table"][b, :-(-kv // PAGE)].long()
    held = torch.uint8 if s["case"]["e4m3"] else torch.bfloat16
    k, v = s["k"].view(held)[at], s["vt"].view(held)[at]
    if s["case"]["e4m3"]:
        k = k.view(torch.float8_e4m3fn).double() * s["k_scale"][at].double()[..., None]
        v = v.view(torch.float8_e4m3fn).double() * s["v_scale"][at].double()[:, :, None]
    k = k.double().permute(1, 0, 2, 3).flatten(1, 2)
    v = v.double().permute(1, 0, 3, 2).flatten(1, 2)
    return k[:, :kv], v[:, :kv]


def _exact_tree(s):
    c = s["case"]
    Hq = c["Hq"]
    G, n0 = Hq // c["Hkv"], 0
    out = torch.zeros(s["N"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["N"], Hq, dtype=torch.float64, device="cuda")
    for b, (ql, kv) in enumerate(_lens(c)):
        k, v = _exact_cache(s, b, kv)
        hidden = np.ones((ql, kv), dtype=bool)
        hidden[:, :kv - ql] = False
        for i in range(ql):
            a = i
            while a >= 0:  # itself and its ancestors
                hidden[i, kv - ql + a] = False
                a = s["parents"][b][a]
        hidden = torch.from_numpy(hidden).cuda()
        for h in range(Hq):
            x = s["q"][n0:n0 + ql, h].double() @ k[h // G].t().contiguous() * math.log(2.0)
            x = x.masked_fill(hidden, -math.inf)
            out[n0:n0 + ql, h] = torch.softmax(x, -1) @ v[h // G]
            lse[n0:n0 + ql, h] = torch.logsumexp(x, -1) / math.log(2.0)
        n0 += ql
    gate = torch.stack([s["proj"][:, h * 2 * D + D:(h + 1) * 2 * D] for h in range(Hq)], 1)
    return (out / (1 + torch.exp(-gate.double()))).reshape(s["N"], Hq * D), lse


def _exact_weights(s):
    c = s["case"]
    G, n0 = c["Hq"] // c["Hkv"], 0
    w = s["weights"].double()
    for b, (ql, kv) in enumerate(_lens(c)):
        k, _ = _exact_cache(s, b, kv)
        at = s["page_table"][b, :-(-kv // PAGE)].long()
        hidden = _behind(kv - ql, ql, kv)
        for kh in range(c["Hkv"]):
            total = s["prev"][at, kh].double().flatten()[:kv].clone()
            total[kv - ql:] = 0
            for h in range(kh * G, kh * G + G):
                x = s["q"][n0:n0 + ql, h].double() @ k[kh].t().contiguous()
                x = torch.exp((x - s["lse"][n0:n0 + ql, h, None].double()) * math.log(2.0))
                total += x.masked_fill(hidden, 0.0).sum(0)
            for i in range(0, kv, PAGE):
                n = min(PAGE, kv - i)
                w[at[i // PAGE], kh, :n] = total[i:i + n]
        n0 += ql
    return w


def _exact_select(s):
    c = s["case"]
    keep, count = s["keep"].cpu().numpy(), s["keep_len"].cpu().numpy()
    table, weights = s["page_table"].tolist(), s["weights"].cpu().numpy()
    for b, (_, kv) in enumerate(_lens(c)):
        n = count[b] = min(kv, c["budget"])
        for h in range(c["Hkv"]):
            chosen = list(range(kv))
            if kv > n:
                lo, hi = c["sinks"], kv - c["recent"]
                w = np.concatenate([weights[p, h] for p in table[b][:-(-kv // PAGE)]])[lo:hi]
                best = np.lexsort((np.arange(hi - lo), -w.astype(np.float64)))
                chosen = list(range(lo)) + list(range(hi, kv)) + \
                    [lo + x for x in best[:n - lo - c["recent"]].tolist()]
            keep[b, h, :n] = sorted(chosen)
    return torch.from_numpy(keep), torch.from_numpy(count)


def _exact_keep(s):
    c = s["case"]
    held = [s["weights"].cpu(), *(s[x].view(torch.uint8 if c["e4m3"] else torch.bfloat16).cpu()
                                  for x in ("k", "vt"))]
    if c["e4m3"]:
        held += [s["k_scale"].cpu(), s["v_scale"].cpu()]
    new = [x.clone() for x in held]
    frm, keep = s["page_table"].tolist(), s["keep"].tolist()
    to = frm if s["to"] is None else s["to"].tolist()
    dst = [0] * c["B"] if s["dst"] is None else s["dst"].tolist()
    for b, n in enumerate(_kept(c)):
        for h in range(c["Hkv"]):
            src = np.array(keep[b][h if len(keep[b]) > 1 else 0][:n])
            goal = np.arange(dst[b], dst[b] + n)
            ps, ss = np.array(frm[b])[src // PAGE], src % PAGE
            pd, sd = np.array(to[b])[goal // PAGE], goal % PAGE
            for x, y in zip(held, new):
                if x.dim() == 4 and x.shape[2] == D:  # V^T: a column
                    y[pd, h, :, sd] = x[ps, h, :, ss]
                else:
                    y[pd, h, sd] = x[ps, h, ss]
    if c["e4m3"]:
        new[1:3] = [x.view(torch.float8_e4m3fn) for x in new[1:3]]
    return new
