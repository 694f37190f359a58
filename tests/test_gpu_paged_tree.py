"""GPU tests of the paged cache's attention of draft trees and of its statistics,
and of rotary positions of several axes, against the float64 forms of
evict_oracle.py and paged_oracle.py (whose bounds are derived there)."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import evict_oracle as eo  # noqa: E402
import paged_oracle as po  # noqa: E402
import test_gpu_paged as gp  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D


def draft(seed, n):
    r = random.Random(seed)
    return [-1 if i == 0 or r.random() < 0.15 else r.randrange(max(0, i - 12), i) for i in range(n)]


def tree_case(seed, Hq, Hkv, e4m3, lens, words=None):
    c = gp.attention_case(seed, Hq, Hkv, e4m3, lens)
    words = words or -(-c["max_q"] // 64)
    rows, c["seen"] = [], []
    for b, (n, _) in enumerate(lens):
        parents = draft(seed + b, n)
        rows += eo.tree_words(parents, words)
        sees = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            a = i
            while a >= 0:
                sees[i, a] = True
                a = parents[a]
        c["seen"].append(sees)
    # rows of no sequence: all bits
    c["tree"] = torch.tensor(rows + [[-1] * words] * (c["N"] - len(rows)), dtype=torch.int64)
    return c


def run(c, tree=None, window=0, sinks=0, gate=True, max_q=None, max_kv=None, want_lse=True):
    o = gp.ops()
    N, Hq = c["N"], c["Hq"]
    max_q, max_kv = max_q or c["max_q"], max_kv or c["max_kv"]
    g = c["gate"].cuda() if gate else None
    out = torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((N, Hq), 7.0, device="cuda") if want_lse else None
    nb = o.attention_paged_ws_bytes(N, len(c["kv_len"]), max_q, max_kv, Hq, c["Hkv"])
    ws = torch.full((nb // 4,), math.nan, device="cuda").view(torch.uint8) if nb else None
    o.attention_paged(c["q"].cuda(), g, Hq * D, D, c["pages"], gp.i32(c["tab"]), gp.i32(c["qs"]),
                      gp.i32(c["kv_len"]), max_q, max_kv, out, window=window, sinks=sinks, ws=ws,
                      tree=None if tree is None else tree.cuda(), lse=lse)
    torch.cuda.synchronize()
    return out.cpu().double().view(N, Hq, D), None if lse is None else lse.cpu().double()


def cache(c, b, kv):
    """K, V [Hkv, kv, D] of sequence b, and which keys are there."""
    k, v = gp.values(c["pages"])
    at = torch.tensor([c["tab"][b][p // PAGE] for p in range(kv)], dtype=torch.long)
    there = (at >= 0) & (at < k.shape[0])
    at, slot = torch.where(there, at, 0), torch.arange(kv) % PAGE
    return k[at, :, slot].transpose(0, 1), v[at, :, slot].transpose(0, 1), there


def check(c, got, lse, seen_of, gate=True, max_q=None):
    """seen_of(b, first row's position, rows, keys): bool [rows, keys]."""
    done = torch.zeros(c["N"], dtype=torch.bool)
    G = c["Hq"] // c["Hkv"]
    for b in range(len(c["kv_len"])):
        q0, ql, p0, kv = eo.rows_of(c, b, max_q)
        K, V, there = cache(c, b, kv)
        seen = seen_of(b, p0, ql, kv) & there
        # values that no row sees may be anything
        for kh in range(c["Hkv"]):
            Vh = torch.where(seen.any(0)[:, None], V[kh], 0.0)
            Kh = torch.where(seen.any(0)[:, None], K[kh], 0.0)
            for h in range(kh * G, kh * G + G):
                rows = slice(q0, q0 + ql)
                ref, tol, rl, tl = eo.attend(c["q"][rows, h].double(), Kh, seen, Vh,
                                             c["gate"][rows, h].double() if gate else None)
                over = (got[rows, h] - ref).abs() - tol
                assert (over <= 0).all(), f"sequence {b} head {h}: {over.max():.3g} over the bound"
                if lse is not None:
                    none = torch.isinf(rl)
                    assert torch.equal(torch.isinf(lse[rows, h]) & (lse[rows, h] < 0), none)
                    over = torch.where(none, -1.0, (lse[rows, h] - rl).abs() - tl)
                    assert (over <= 0).all(), f"lse of sequence {b} head {h}: {over.max():.3g} over"
        done[q0:q0 + ql] = True
    assert (got[~done] == 7.0).all(), "rows of no sequence were written"
    if lse is not None:
        assert (lse[~done] == 7.0).all()


def tree_seen(c):
    def f(b, p0, ql, kv):
        seen = torch.ones(ql, kv, dtype=torch.bool)
        lo = max(p0, 0)
        seen[:, lo:] = c["seen"][b][:ql, lo - p0:kv - p0]
        return seen
    return f


def causal(window=0, sinks=0):
    def f(b, p0, ql, kv):
        p, j = torch.arange(p0, p0 + ql)[:, None], torch.arange(kv)
        seen = j <= p
        return seen & ((j > p - window) | (j < sinks)) if window else seen
    return f


TREES = [
    # (Hq, Hkv, [(drafted tokens, keys)])
    (8, 2, [(1, 1)]),
    (8, 2, [(4, 300)]),                                     # few rows, in parts
    (16, 4, [(3, 3), (4, 64), (2, 65), (1, 700), (0, 70), (4, 130)]),
    (16, 4, [(26, 530)]),
    (4, 1, [(5, 3), (64, 128), (3, 66), (63, 63)]),          # fewer keys than tokens
    (8, 2, [(64, 64), (40, 1500), (33, 97), (0, 5), (1, 64)]),
    (4, 4, [(65, 70), (130, 1000), (64, 65)]),               # more words than one
    (16, 1, [(200, 333), (7, 450)]),
    (6, 2, [(17, 80)] * 70),                                 # more than 64 sequences
    (16, 2, [(2, 63)] * 70 + [(0, 9)] * 5),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", TREES)
def test_trees_match_oracle(Hq, Hkv, lens, e4m3):
    c = tree_case(301, Hq, Hkv, e4m3, lens)
    got, lse = run(c, c["tree"])
    check(c, got, lse, tree_seen(c))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(3, 700), (2, 64)], [(40, 700), (33, 97)]])
def test_trees_without_gate_lse_and_with_loose_bounds(lens, e4m3):
    """More words than needed, larger max_q and max_kv; lse not asked for gives the
    same bits."""
    c = tree_case(311, 8, 2, e4m3, lens, words=3)
    for row in c["tab"]:
        row += [-1] * 5
    got, lse = run(c, c["tree"], gate=False, max_q=150, max_kv=16 * PAGE)
    check(c, got, lse, tree_seen(c), gate=False)
    again, _ = run(c, c["tree"], gate=False, max_q=150, max_kv=16 * PAGE, want_lse=False)
    assert torch.equal(got, again)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(4, 300), (3, 100)], [(60, 300), (70, 1500)]])
def test_a_chain_has_the_bits_of_causal_attention(lens, e4m3):
    """A tree of one branch is what the causal call computes; its lse call gives the bits
    of the call without."""
    c = tree_case(321, 16, 4, e4m3, lens)
    words = c["tree"].shape[1]
    rows = [r for n, _ in lens for r in eo.tree_words(list(range(-1, n - 1)), words)]
    chain = torch.tensor(rows + [[0] * words] * (c["N"] - len(rows)), dtype=torch.int64)
    got, lse = run(c, chain)
    check(c, got, lse, causal())
    out, lse2 = run(c)
    check(c, out, lse2, causal())
    plain, _ = run(c, want_lse=False)
    assert torch.equal(out, plain)
    if max(n for n, _ in lens) <= 4:  # few rows: every unit's keys are the same ones
        assert torch.equal(got, plain) and torch.equal(lse, lse2)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (100, 4), (64, 70)])
@pytest.mark.parametrize("Hq,Hkv,lens", [
    (16, 4, [(1, 700), (1, 64), (1, 1), (0, 9), (3, 130)]), (8, 2, [(60, 700), (5, 3), (33, 97)]),
    (4, 1, [(1, 3000)]), (4, 1, [(300, 3000)])])
def test_lse_of_causal_calls(Hq, Hkv, lens, window, sinks, e4m3):
    c = gp.attention_case(331, Hq, Hkv, e4m3, lens)
    got, lse = run(c, window=window, sinks=sinks)
    check(c, got, lse, causal(window, sinks))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(3, 300), (4, 64), (2, 130)], [(40, 300), (33, 97), (20, 20)]])
def test_trees_ignore_what_no_row_sees(lens, e4m3):
    """Nodes cut off from every row (no bit, not even their own), keys behind the last
    and foreign pages hold NaN in K, V and scales: no result has any of it."""
    c = tree_case(341, 8, 2, e4m3, lens)
    pages = c["pages"]
    used = torch.zeros(pages.num_pages, PAGE, dtype=torch.bool)
    for b, (n, kv) in enumerate(lens):
        q0 = c["qs"][b]
        for i in range(n):  # node 1 and every node below it see all but node 1
            c["seen"][b][i, 1] = False
            c["tree"][q0 + i, 0] &= ~2
        for p in range(kv):
            if p != kv - n + 1:
                used[c["tab"][b][p // PAGE], p % PAGE] = True
    bad = ~used.cuda()
    nan = 0x7f if e4m3 else 0x7fc0
    raw = (lambda t: t.view(torch.uint8)) if e4m3 else (lambda t: t.view(torch.int16))
    raw(pages.k).masked_fill_(bad[:, None, :, None], nan)
    raw(pages.vt).masked_fill_(bad[:, None, None, :], nan)
    if e4m3:
        pages.k_scale.masked_fill_(bad[:, None], math.nan)
        pages.v_scale.masked_fill_(bad[:, None], math.inf)
    got, lse = run(c, c["tree"])
    assert torch.isfinite(got).all()
    check(c, got, lse, tree_seen(c))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(3, 3), (2, 2)], [(30, 30), (70, 70), (64, 100)]])
def test_rows_that_see_nothing_give_zero(lens, e4m3):
    c = tree_case(351, 8, 2, e4m3, lens)
    for b, (n, kv) in enumerate(lens):
        for i in range(0, n, 2):
            c["seen"][b][i] = False
            c["tree"][c["qs"][b] + i] = 0
    got, lse = run(c, c["tree"])
    check(c, got, lse, tree_seen(c))
    assert (got[0] == 0).all() and torch.isinf(lse[0]).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(4, 400), (3, 90)], [(40, 400), (3, 70)]])
def test_trees_skip_pages_that_are_not_there(lens, e4m3):
    c = tree_case(361, 8, 2, e4m3, lens)
    c["tab"][0][2], c["tab"][1][1] = -1, c["pages"].num_pages
    got, lse = run(c, c["tree"])
    check(c, got, lse, tree_seen(c))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,max_q", [([(8, 300), (2, 90), (5, 64)], 3),
                                        ([(80, 300), (2, 90), (65, 128)], 50)])
def test_trees_past_max_q(lens, max_q, e4m3):
    """Rows past max_q are left alone, and their keys seen by none."""
    c = tree_case(371, 8, 2, e4m3, lens)
    got, lse = run(c, c["tree"], max_q=max_q)
    check(c, got, lse, tree_seen(c), max_q=max_q)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(4, 300), (3, 70)], [(40, 300), (70, 90)]])
@pytest.mark.parametrize("scale", [900.0, -900.0])
def test_trees_of_large_scores(lens, scale, e4m3):
    c = tree_case(381, 8, 2, e4m3, lens)
    c["q"] = (c["q"].float() * abs(scale)).bfloat16() * (1 if scale > 0 else -1)
    got, lse = run(c, c["tree"])
    check(c, got, lse, tree_seen(c))


def test_trees_captured_on_a_stream_and_replayed():
    """Lengths, tables, masks and values change between replays of one graph."""
    o = gp.ops()
    Hq, Hkv = 8, 2
    a = tree_case(391, Hq, Hkv, True, [(20, 400), (9, 70)])
    b = tree_case(394, Hq, Hkv, True, [(8, 130), (21, 300)])
    st = dict(q=a["q"].cuda(), tab=gp.i32(a["tab"]), qs=gp.i32(a["qs"]),
              kv=gp.i32(a["kv_len"]), tree=a["tree"].cuda())
    out = torch.zeros(a["N"], Hq * D, dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros(a["N"], Hq, device="cuda")
    nb = o.attention_paged_ws_bytes(a["N"], 2, 32, 448, Hq, Hkv)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None

    def step():
        o.attention_paged(st["q"], None, 0, 0, a["pages"], st["tab"], st["qs"], st["kv"], 32, 448,
                          out, ws=ws, tree=st["tree"], lse=lse)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    b["pages"] = a["pages"]
    b["tab"] = [[x % a["pages"].num_pages if x >= 0 else x for x in r] for r in b["tab"]]
    width = st["tab"].shape[1]
    b["tab"] = [(r + [-1] * width)[:width] for r in b["tab"]]
    for c in (a, b, a, b):
        st["q"].copy_(c["q"])
        st["tab"].copy_(torch.tensor(c["tab"], dtype=torch.int32))
        st["qs"].copy_(torch.tensor(c["qs"], dtype=torch.int32))
        st["kv"].copy_(torch.tensor(c["kv_len"], dtype=torch.int32))
        st["tree"].copy_(c["tree"])
        out.fill_(7.0), lse.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(c, out.cpu().double().view(-1, Hq, D), lse.cpu().double(), tree_seen(c), gate=False)
        want = out.clone()
        out.fill_(7.0)
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- rotary positions of several axes ------------------------------------------------
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rot,axis_of", [
    (64, [i % 3 if i % 3 and i < 30 else 0 for i in range(32)]), (64, [0] * 16 + [1] * 16),
    (64, [0] * 31 + [3]), (32, [0, 1, 2, 3] * 4), (16, [2] * 8), (8, [1, 0, 1, 0]), (32, [0] * 16),
    (16, [0] * 8), (8, [0] * 4)])
@pytest.mark.parametrize("Hq,Hkv,lens", [
    (16, 4, [(37, 37), (0, 0), (16, 80), (1, 97)]), (6, 1, [(5, 3), (3, 66)]),
    (4, 2, [(1, 3), (0, 5), (2, 66)] * 40)])
def test_prep_of_several_axes(Hq, Hkv, lens, rot, axis_of, e4m3):
    """q and K against the 64-bit form (one rounding; of fp32's arithmetic 1e-5 of the
    row's largest), e4m3 keys that form's own bytes; V the bits of the one-axis call."""
    o = gp.ops()
    q_lens, kv_len = [n for n, _ in lens], [k for _, k in lens]
    qs, N = gp.starts(q_lens), sum(q_lens) + 2
    num_pages = sum(-(-k // PAGE) for k in kv_len) + 2
    pages, plain = gp.pool(401, num_pages, Hkv, e4m3), gp.pool(401, num_pages, Hkv, e4m3)
    tab = gp.table(402, kv_len, num_pages)
    g = torch.Generator().manual_seed(403)
    width = Hq * 512 + Hkv * 512
    proj = torch.randn(N, width, generator=g).bfloat16()
    qw, kw = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    axes = o.RopeAxes(axis_of)
    pos = torch.randint(0, 700, (axes.axes, N), generator=g, dtype=torch.int32)
    rope = o.rope_table(1e7, rot, 700)
    q_out = torch.full((N, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")

    def prep(p, into, q, **kw_):
        o.attn_prep_paged(proj.cuda(), qw.cuda(), kw.cuda(), p.cuda(), gp.i32(qs), gp.i32(kv_len),
                          gp.i32(tab), Hq, rot, rope, 1e-6, gp.Q_SCALE, q, into, **kw_)

    prep(pos, pages, q_out, axes=axes)
    prep(pos[0].contiguous(), plain, torch.empty_like(q_out))
    torch.cuda.synchronize()
    raw = lambda t: t.view(torch.uint8 if e4m3 else torch.int16)
    assert torch.equal(raw(pages.vt), raw(plain.vt))
    table = rope.cpu().double()
    cs = torch.stack([table[pos[a].long(), i] for i, a in enumerate(axis_of)], 1)[:, None]
    x = proj.double()
    q = po.norm_rope(x[:, :Hq * 512].view(-1, Hq, 512)[..., :D], qw.double(), cs[..., 0],
                     cs[..., 1], rot, 1e-6) * gp.Q_SCALE
    k = po.norm_rope(x[:, Hq * 512:Hq * 512 + Hkv * 256].view(-1, Hkv, D), kw.double(),
                     cs[..., 0], cs[..., 1], rot, 1e-6)
    n, got = qs[-1], q_out.cpu().double()
    assert ((got - q)[:n].abs() <= q[:n].abs() * 2 ** -8 +
            1e-5 * q[:n].abs().amax(-1, keepdim=True)).all()
    assert (got[n:] == 7.0).all()
    gk = pages.k.cpu().float().double()
    for b in range(len(lens)):
        for r, _, page, slot in po.slots(qs, kv_len, tab, b, num_pages):
            if e4m3:
                kq, ks = po.quantise(k[r], 1)
                assert torch.equal(pages.k_scale[page, :, slot].cpu().double(), ks), (b, r)
                assert torch.equal(gk[page, :, slot], kq), (b, r)
            else:
                bound = k[r].abs() * 2 ** -8 + 1e-5 * k[r].abs().amax(1, keepdim=True)
                assert ((gk[page, :, slot] - k[r]).abs() <= bound).all(), (b, r)


@pytest.mark.parametrize("e4m3", [False, True])
def test_axes_with_the_same_positions_have_the_bits_of_one(e4m3):
    o = gp.ops()
    Hq, Hkv, N = 8, 2, 50
    a, b = gp.pool(411, 3, Hkv, e4m3), gp.pool(411, 3, Hkv, e4m3)
    g = torch.Generator().manual_seed(412)
    proj = torch.randn(N, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    w = (1 + 0.1 * torch.randn(D, generator=g)).cuda()
    pos = torch.randint(-3, 300, (N,), generator=g, dtype=torch.int32).cuda()  # cut to the table
    rope = o.rope_table(1e7, 64, 250)
    outs = []
    for pages, p, axes in ((a, pos, None),
                           (b, pos.repeat(3, 1), o.RopeAxes.from_sections([11, 11, 10], True))):
        q = torch.zeros(N, Hq, D, dtype=torch.bfloat16, device="cuda")
        o.attn_prep_paged(proj, w, w, p, gp.i32([0, N]), gp.i32([N + 7]), gp.i32([[2, 0]]), Hq, 64,
                          rope, 1e-6, gp.Q_SCALE, q, pages, axes=axes)
        outs += [q, pages.k.view(torch.uint8), pages.vt.view(torch.uint8)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[:3], outs[3:]))
