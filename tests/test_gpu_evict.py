"""GPU tests of eviction from the paged cache against the float64 forms of
evict_oracle.py (whose bounds are derived there): weights by key, positions to keep
(exact), their move (exact), and a run of all with the attention around them."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import evict_oracle as eo  # noqa: E402
import paged_oracle as po  # noqa: E402
import test_gpu_paged as gp  # noqa: E402
import test_gpu_paged_tree as gt  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D


# ---- weights by key ---------------------------------------------------------------
def fill(c, seed):
    """prev and weights that hold something everywhere, and lse of the call's rows (about
    what the attention gives; the rows of no sequence hold NaN)."""
    g = torch.Generator().manual_seed(seed)
    shape = (c["pages"].num_pages, c["Hkv"], PAGE)
    c["prev"], c["w"] = torch.rand(*shape, generator=g), torch.rand(*shape, generator=g)
    c["lse"] = torch.full((c["N"], c["Hq"]), math.nan)
    G = c["Hq"] // c["Hkv"]
    for b in range(len(c["kv_len"])):
        q0, ql, p0, kv = eo.rows_of(c, b)
        K, _, there = gt.cache(c, b, kv)
        seen = gt.causal()(b, p0, ql, kv) & there
        K = torch.where(seen.any(0)[:, None], K, 0.0)
        for h in range(c["Hq"]):
            c["lse"][q0:q0 + ql, h] = eo.attend(c["q"][q0:q0 + ql, h].double(), K[h // G],
                                                seen)[0].float()
    return c


def weigh(c, prev="prev", max_q=None, max_kv=None):
    o = gp.ops()
    w = c["w"].cuda()
    p = {"prev": c["prev"].cuda(), "in place": w, None: None}[prev]
    o.kv_weights(c["q"].cuda(), c["lse"].cuda(), c["pages"], gp.i32(c["tab"]), gp.i32(c["qs"]),
                 gp.i32(c["kv_len"]), max_q or c["max_q"], max_kv or c["max_kv"], w, prev=p)
    torch.cuda.synchronize()
    return w.cpu()


def check_weights(c, got, prev="prev", max_q=None, max_kv=None):
    G, want = c["Hq"] // c["Hkv"], c["w"].clone().double()
    tol = torch.zeros_like(want)
    before = {"prev": c["prev"], "in place": c["w"], None: torch.zeros_like(c["w"])}[prev].double()
    for b in range(len(c["kv_len"])):
        q0, ql, p0, kv = eo.rows_of(c, b, max_q)
        kv = min(kv, max_kv or kv)
        if ql <= 0 or kv <= 0:
            continue
        K, _, there = gt.cache(c, b, kv)
        seen = gt.causal()(b, p0, ql, kv) & there
        K = torch.where(seen.any(0)[:, None], K, 0.0)
        for kh in range(c["Hkv"]):
            heads = slice(kh * G, kh * G + G)
            w, t = eo.weights(c["q"][q0:q0 + ql, heads].double(),
                              c["lse"][q0:q0 + ql, heads].double(), K[kh], seen)
            for p in range(kv):
                page = c["tab"][b][p // PAGE]
                if not there[p]:
                    continue
                add = before[page, kh, p % PAGE] if p < p0 else 0.0
                want[page, kh, p % PAGE] = w[p] + add
                tol[page, kh, p % PAGE] = t[p] + 2.0 ** -23 * abs(add)
    over = (got.double() - want).abs() - tol
    assert not torch.isnan(over).any()
    assert (over <= 0).all(), f"off by {over.max():.3g} over the bound, at {int(over.argmax())}"


WEIGHTS = [
    # (Hq, Hkv, [(new tokens, keys)])
    (8, 2, [(1, 1)]),
    (16, 4, [(1, 1), (1, 64), (1, 65), (0, 70), (1, 300), (3, 130)]),
    (4, 1, [(1, 1500)]),
    (4, 4, [(40, 40), (33, 900), (1, 513)]),
    (8, 2, [(70, 70), (200, 700)]),
    (4, 1, [(5, 3), (64, 128), (130, 66)]),      # fewer keys than tokens
    (16, 4, [(530, 530)]),
    (16, 1, [(100, 612)]),
    (6, 2, [(17, 300)] * 40),                     # a page a wave: many workgroups
    (16, 4, [(2, 600)] * 70 + [(0, 5)] * 3),
    (7, 1, [(50, 1100)]),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", WEIGHTS)
def test_weights_match_oracle(Hq, Hkv, lens, e4m3):
    c = fill(gp.attention_case(601, Hq, Hkv, e4m3, lens), 602)
    check_weights(c, weigh(c))


@pytest.mark.parametrize("prev", [None, "in place"])
@pytest.mark.parametrize("lens", [[(1, 300), (2, 64)], [(60, 300), (33, 97)]])
def test_weights_anew_and_in_place(lens, prev):
    c = fill(gp.attention_case(611, 8, 2, True, lens), 612)
    check_weights(c, weigh(c, prev), prev)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(1, 300), (2, 70)], [(60, 300), (33, 97)]])
def test_weights_of_slots_and_rows_that_hold_anything(lens, e4m3):
    """NaN in K, its scales, prev and weights past the last key and in foreign pages, a
    row whose lse is -inf, one page that is not there, loose bounds."""
    c = gp.attention_case(621, 8, 2, e4m3, lens)
    pages = c["pages"]
    used = torch.zeros(pages.num_pages, PAGE, dtype=torch.bool)
    for b, (n, kv) in enumerate(lens):
        for p in range(kv):
            used[c["tab"][b][p // PAGE], p % PAGE] = True
    c["tab"][0][1] = -5
    bad = ~used.cuda()
    raw = (lambda t: t.view(torch.uint8)) if e4m3 else (lambda t: t.view(torch.int16))
    raw(pages.k).masked_fill_(bad[:, None, :, None], 0x7f if e4m3 else 0x7fc0)
    if e4m3:
        pages.k_scale.masked_fill_(bad[:, None], math.nan)
    c = fill(c, 622)
    c["lse"][c["qs"][1]] = -math.inf
    for name in ("prev", "w"):
        c[name] = torch.where(used[:, None], c[name], 7.0)
    c["prev"] = torch.where(used[:, None], c["prev"], math.nan)
    for row in c["tab"]:
        row += [-1] * 3
    check_weights(c, weigh(c, max_q=100, max_kv=8 * PAGE))


@pytest.mark.parametrize("lens,max_q,max_kv", [([(8, 300), (2, 90)], 3, None),
                                               ([(80, 300), (2, 90)], 50, None),
                                               ([(8, 300), (2, 90)], 8, 100),
                                               ([(80, 300), (20, 90)], 80, 130)])
def test_weights_past_max_q_and_max_kv(lens, max_q, max_kv):
    c = fill(gp.attention_case(631, 8, 2, False, lens), 632)
    check_weights(c, weigh(c, max_q=max_q, max_kv=max_kv), max_q=max_q, max_kv=max_kv)


def test_weights_with_a_bound_far_past_the_keys():
    """Tables of 2^20 columns, for which a wave takes more pages than one."""
    c = fill(gp.attention_case(636, 8, 4, True, [(2, 700), (1, 130)]), 637)
    want = weigh(c)
    wide = [row + [-1] * ((1 << 20) - len(row)) for row in c["tab"]]
    got = weigh({**c, "tab": wide}, max_kv=1 << 26)
    assert torch.equal(got, want)


def test_weights_repeat_bit_for_bit_on_any_stream():
    c = fill(gp.attention_case(641, 16, 4, True, [(300, 700), (33, 97), (1, 64)]), 642)
    first = weigh(c)
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            assert torch.equal(weigh(c), first)


@pytest.mark.parametrize("e4m3", [False, True])
def test_weights_of_large_scores(e4m3):
    """Peaked rows: one key has nearly all of a row's weight."""
    c = gp.attention_case(651, 8, 2, e4m3, [(50, 300), (1, 70)])
    c["q"] = (c["q"].float() * 60).bfloat16()
    c = fill(c, 652)
    check_weights(c, weigh(c))


# ---- positions to keep -----------------------------------------------------------------
def select_case(seed, Hkv, kv_len, kind):
    need = [-(-max(k, 0) // PAGE) for k in kv_len]
    num_pages = sum(need) + 2
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2 * torch.randn(num_pages, Hkv, PAGE, generator=g))
    if kind == "ties":
        w = torch.round(w)
    elif kind == "same":
        w.fill_(0.25)
    elif kind == "any":  # all of the type's values
        w = torch.randint(-2 ** 31, 2 ** 31, w.shape, generator=g).int().view(torch.float32)
        w[..., ::7], w[..., 1::7] = 0.0, -0.0
    return w, gp.table(seed + 1, kv_len, num_pages), num_pages


@pytest.mark.parametrize("kind", ["spread", "ties", "same", "any"])
@pytest.mark.parametrize("Hkv,kv_len,budget,sinks,recent", [
    (2, [1, 0, 64, 65, 300], 40, 4, 10),
    (1, [700], 1, 0, 0), (1, [700], 1, 1, 0), (1, [700], 1, 0, 1), (1, [700], 699, 4, 64),
    (4, [1500, 1024, 1025, 90], 512, 0, 0), (4, [900, 33], 100, 60, 40),
    (1, [5000, 4096, 4097], 2500, 4, 256), (2, [10000], 3000, 4, 100),
    (1, [20000, 17000, 3], 9000, 4, 1000), (3, [130] * 70, 65, 1, 1), (2, [50, 60], 0, 0, 0)])
def test_select_matches_oracle(Hkv, kv_len, budget, sinks, recent, kind):
    o = gp.ops()
    w, tab, _ = select_case(701, Hkv, kv_len, kind)
    B, max_kv = len(kv_len), max(kv_len)
    keep = torch.full((B, Hkv, budget + 3), -7, dtype=torch.int32, device="cuda")
    n = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    o.kv_select(w.cuda(), gp.i32(tab), gp.i32(kv_len), max_kv, budget, keep, n, sinks=sinks,
                recent=recent)
    torch.cuda.synchronize()
    keep, n = keep.cpu(), n.tolist()
    for b, kv in enumerate(kv_len):
        assert n[b] == min(kv, budget)
        for h in range(Hkv):
            at = [w[p, h] for p in tab[b] if p >= 0]
            ws = torch.cat(at).tolist() if at else []
            assert keep[b, h, :n[b]].tolist() == eo.select(ws, kv, budget, sinks, recent), (b, h)
            assert (keep[b, h, n[b]:] == -7).all()


def test_select_puts_missing_pages_last_and_cuts_lengths():
    """Pages outside the pool are the lightest, below weights of -inf; lengths past max_kv
    and below 0 are cut."""
    o = gp.ops()
    w, tab, num_pages = select_case(711, 2, [300, 300, 300, 300], "spread")
    tab[0][1], tab[0][3], tab[1][0] = -1, num_pages, 2 ** 31 - 1
    w[tab[0][0]] = -math.inf
    keep = torch.full((4, 2, 150), -7, dtype=torch.int32, device="cuda")
    n = torch.zeros(4, dtype=torch.int32, device="cuda")
    o.kv_select(w.cuda(), gp.i32(tab), gp.i32([300, 280, 10 ** 9, -4]), 290, 150, keep, n, sinks=2,
                recent=30)
    torch.cuda.synchronize()
    assert n.tolist() == [150, 150, 150, 0]
    for b, kv in enumerate([290, 280, 290]):
        for h in range(2):
            ws = []
            for p in tab[b]:
                ws += w[p, h].tolist() if 0 <= p < num_pages else [None] * PAGE
            assert keep[b, h].tolist() == eo.select(ws, kv, 150, 2, 30), (b, h)
    assert (keep[3] == -7).all()


# ---- their move --------------------------------------------------------------------------
def moved(pages, w, tab, keep, n, dst=None, to=None):
    """(k, vt, scales..., w) bytes on the CPU, moved one by one from a copy."""
    raw = lambda t: t.view(torch.uint8 if t.itemsize == 1 else torch.int16 if t.itemsize == 2
                           else torch.int32).cpu()
    old = [raw(pages.k), raw(pages.vt).transpose(2, 3)]
    old += [raw(t) for t in (pages.k_scale, pages.v_scale, w) if t is not None]
    new = [t.clone() for t in old]
    to = tab if to is None else to
    inside = lambda t, b, p: 0 <= p < len(t[b]) * PAGE and 0 <= t[b][p // PAGE] < pages.num_pages
    for b in range(len(tab)):
        for h in range(pages.Hkv):
            row = keep[b][h if len(keep[b]) > 1 else 0]
            for i in range(min(n[b], len(row))):
                p, d = row[i], (dst[b] if dst else 0) + i
                if inside(tab, b, p) and inside(to, b, d):
                    for a, z in zip(old, new):
                        z[to[b][d // PAGE], h, d % PAGE] = a[tab[b][p // PAGE], h, p % PAGE]
    return new


def keep_and_check(pages, w, tab, keep, n, dst=None, to=None):
    o = gp.ops()
    want = moved(pages, w, tab, keep, n, dst, to)
    o.kv_keep(pages, gp.i32(tab), gp.i32(keep), gp.i32(n), dst=None if dst is None else gp.i32(dst),
              to_table=None if to is None else gp.i32(to), weights=w)
    torch.cuda.synchronize()
    raw = lambda t: t.view(torch.uint8 if t.itemsize == 1 else torch.int16 if t.itemsize == 2
                           else torch.int32).cpu()
    got = [raw(pages.k), raw(pages.vt).transpose(2, 3)]
    got += [raw(t) for t in (pages.k_scale, pages.v_scale, w) if t is not None]
    for name, a, b in zip(("k", "vt", "k_scale", "v_scale", "weights"), got, want):
        assert torch.equal(a, b), name


def lists(seed, kv_len, heads, most):
    r = random.Random(seed)
    n = [min(k, r.randint(0, most)) if i else min(k, most) for i, k in enumerate(kv_len)]
    keep = [[sorted(r.sample(range(k), m)) + [-1] * (most - m) for _ in range(heads)]
            for k, m in zip(kv_len, n)]
    return keep, n


KEEPS = [(2, [1, 0, 64, 65, 300], 40), (4, [700, 530], 300), (1, [3000], 1500), (2, [2100], 2100),
         (1, [100] * 70, 20), (3, [257, 600, 33], 257)]


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("Hkv,kv_len,most", KEEPS)
def test_keep_in_place(Hkv, kv_len, most, one, e4m3, weighted):
    num_pages = sum(-(-k // PAGE) for k in kv_len) + 2
    pages = gp.pool(801, num_pages, Hkv, e4m3)
    w = torch.rand(num_pages, Hkv, PAGE, device="cuda") if weighted else None
    keep, n = lists(802, kv_len, 1 if one else Hkv, most)
    keep_and_check(pages, w, gp.table(803, kv_len, num_pages), keep, n)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hkv,kv_len,most", KEEPS)
def test_keep_into_other_pages(Hkv, kv_len, most, e4m3):
    """Lists in any order, with repeats."""
    r = random.Random(811)
    need = [-(-k // PAGE) for k in kv_len]
    per = -(-most // PAGE)
    num_pages = sum(need) + len(kv_len) * per
    pages = gp.pool(812, num_pages, Hkv, e4m3)
    w = torch.rand(num_pages, Hkv, PAGE, device="cuda")
    tab = gp.table(813, kv_len, num_pages)
    left = [p for p in range(num_pages) if p not in {x for row in tab for x in row}]
    to = [[left.pop() for _ in range(per)] for _ in kv_len]
    n = [min(most, k) for k in kv_len]
    keep = [[[r.randrange(k) if k else 0 for _ in range(most)] for _ in range(Hkv)] for k in kv_len]
    keep_and_check(pages, w, tab, keep, n, to=to)


@pytest.mark.parametrize("e4m3", [False, True])
def test_keep_of_accepted_paths(e4m3):
    """Paths of draft trees move to the first places behind the committed keys, across the
    ends of pages; some are where they go already."""
    r = random.Random(821)
    committed, T = [60, 0, 63, 64, 500, 129], 30
    kv_len = [k + T for k in committed]
    num_pages = sum(-(-k // PAGE) for k in kv_len) + 2
    pages = gp.pool(822, num_pages, 2, e4m3)
    n = [5, 7, 1, 0, 30, 8]
    keep = [[[k + x for x in sorted(r.sample(range(T), m))] + [0] * (30 - m)]
            for k, m in zip(committed, n)]
    keep_and_check(pages, None, gp.table(823, kv_len, num_pages), keep, n, dst=committed)


@pytest.mark.parametrize("to", [False, True])
def test_keep_leaves_out_what_is_nowhere(to):
    """Sources and goals outside the tables and pages outside the pool move nothing;
    counts past the list are cut, negative ones are none."""
    kv_len = [200, 200, 200, 200]
    pages = gp.pool(831, 20, 2, True)
    w = torch.rand(20, 2, PAGE, device="cuda")
    tab = gp.table(832, kv_len, 20)
    tab[0][0], tab[1][1] = 20, -1
    keep = [[list(range(3, 143))] * 2 for _ in range(4)]
    keep[2] = [[-1, 5, 2 ** 31 - 1, 256, 100, -2 ** 31] + [150] * 134] * 2
    left = [p for p in range(20) if p not in {x for row in tab for x in row}]
    other = [[left[0], -3], [20, left[1]], [left[2], left[3]], [0, 0]] if to else None
    n = [140, 10 ** 9, 140, -5]
    dst = [0, 0, 0, 0] if to else [0, -3, 250, 1]
    if not to:  # the third's goals leave the table; its list ascends from there
        keep[2] = [[250, 251, 252, 255, 256, 300] + [400] * 134] * 2
    keep_and_check(pages, w, tab, keep, n, dst=dst, to=other)


# ---- together ------------------------------------------------------------------------------
@pytest.mark.parametrize("e4m3", [False, True])
def test_a_served_sequence_from_prompt_to_accepted_draft(e4m3):
    """Two sequences, as a server runs them on one stream: a prompt with pictures' axes
    is written and attended with its statistics, its weights select what each kv-head
    keeps, the rest is evicted in place, tokens are decoded on what is left with their
    weights added, a draft tree is attended, its accepted path moved into place, and a
    further token decoded. Every output against float64 on the keys that each step has."""
    o = gp.ops()
    Hq, Hkv, rot = 8, 2, 64
    G, lens = Hq // Hkv, [330, 150]
    budget, sinks, recent = 100, 4, 32
    pages = gp.pool(901, 14, Hkv, e4m3)
    tab = gp.table(902, [400, 400], 14)
    g = torch.Generator().manual_seed(903)
    qw, kw = (1 + 0.1 * torch.randn(D, generator=g)).cuda(), (1 + 0.1 * torch.randn(D, generator=g)).cuda()
    rope, axes = o.rope_table(1e7, rot, 1000), o.RopeAxes.from_sections([11, 11, 10], True)
    w = torch.rand(14, Hkv, PAGE, device="cuda")
    ws = torch.empty(o.attention_paged_ws_bytes(480, 2, 330, 448, Hq, Hkv), dtype=torch.uint8,
                     device="cuda")
    kv = [0, 0]  # keys that are kept
    t32 = gp.i32(tab)

    def step(new, pos, parents=None, weigh=None):
        """new tokens a sequence; pos [3][N]. Writes, attends, checks; gives lse."""
        nonlocal kv
        N, qs = sum(new), gp.starts(new)
        kv = [a + b for a, b in zip(kv, new)]
        proj = (torch.randn(N, Hq * 512 + Hkv * 512, generator=g) * 1.5).bfloat16()
        q = torch.zeros(N, Hq, D, dtype=torch.bfloat16, device="cuda")
        out = torch.zeros(N, Hq * D, dtype=torch.bfloat16, device="cuda")
        lse = torch.zeros(N, Hq, device="cuda")
        gate = proj.cuda()
        words = -(-max(new) // 64)
        tree = None if parents is None else torch.tensor(
            [x for p in parents for x in eo.tree_words(p, words)], dtype=torch.int64).cuda()
        o.attn_prep_paged(gate, qw, kw, gp.i32(pos), gp.i32(qs), gp.i32(kv), t32, Hq, rot, rope,
                          1e-6, gp.Q_SCALE, q, pages, axes=axes)
        o.attention_paged(q, gate[:, D:], gate.stride(0), 2 * D, pages, t32, gp.i32(qs), gp.i32(kv),
                          max(new), 448, out, ws=ws, tree=tree, lse=lse)
        before = w.clone()
        if weigh is not None:
            o.kv_weights(q, lse, pages, t32, gp.i32(qs), gp.i32(kv), max(new), 448, w, prev=weigh)
        torch.cuda.synchronize()
        c = dict(pages=pages, tab=tab, q=q.cpu(), qs=qs, kv_len=list(kv), N=N, Hq=Hq, Hkv=Hkv,
                 max_q=max(new), gate=proj[:, :Hq * 512].view(N, Hq, 2, D)[:, :, 1].contiguous(),
                 seen=[])
        seen = gt.causal()
        if parents is not None:
            for p in parents:
                s = torch.eye(len(p), dtype=torch.bool)
                for i, a in enumerate(p):
                    if a >= 0:
                        s[i] |= s[a]
                c["seen"].append(s)
            seen = gt.tree_seen(c)
        gt.check(c, out.cpu().double().view(N, Hq, D), lse.cpu().double(), seen)
        if weigh is not None:
            c.update(lse=lse.cpu(), w=before.cpu(), prev=before.cpu(), max_kv=448)
            check_weights(c, w.cpu(), "in place" if weigh is w else None)
        return c

    # a prompt: text, then a picture's patches in rows and columns, then text
    pos = [[], [], []]
    for n in lens:
        for i in range(n):
            pic = 40 <= i < 120
            at = i if i < 40 else i - 70
            for a, p in enumerate((40, 40 + (i - 40) // 10, 40 + (i - 40) % 10) if pic else (at,) * 3):
                pos[a].append(p)
    step(lens, pos)
    # the last 16 tokens' weights (a call with those rows alone) select what stays
    last = [16, 16]
    kv = [k - 16 for k in kv]
    step(last, [[300 + i % 16 for i in range(32)]] * 3)
    kv = [k - 16 for k in kv]
    w.zero_()
    step(last, [[300 + i % 16 for i in range(32)]] * 3, weigh=w)
    keep = torch.zeros(2, Hkv, budget, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    o.kv_select(w, t32, gp.i32(kv), 448, budget, keep, n, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    held = w.cpu()
    for b in range(2):
        for h in range(Hkv):
            ws_ = torch.cat([held[p, h] for p in tab[b] if p >= 0]).tolist()
            assert keep[b, h].tolist() == eo.select(ws_, kv[b], budget, sinks, recent)
    keep_and_check(pages, w, tab, keep.tolist(), n.tolist())
    kv = n.tolist()
    for t in range(2):
        step([1, 1], [[500 + t] * 2] * 3, weigh=w)
    parents = [gt.draft(904, 20), gt.draft(905, 9)]
    step([20, 9], [[502 + i % 5 for i in range(29)]] * 3, parents=parents)
    # accept a path of each: from its deepest node up
    paths = []
    for p in parents:
        path, a = [], len(p) - 1
        while a >= 0:
            path.append(a)
            a = p[a]
        paths.append(path[::-1])
    base = [k - len(p) for k, p in zip(kv, parents)]
    most = max(map(len, paths))
    keep_and_check(pages, w, tab, [[[k + x for x in p] + [0] * (most - len(p))]
                                   for k, p in zip(base, paths)], [len(p) for p in paths], dst=base)
    kv = [k + len(p) for k, p in zip(base, paths)]
    step([1, 1], [[510] * 2] * 3, weigh=w)


def test_a_captured_eviction_replays_with_other_lengths():
    """Weights, selection and move in one graph, replayed over other lengths, tables and
    values, with eager work between; each against the eager calls on a copy."""
    o = gp.ops()
    Hq, Hkv, budget, num_pages = 8, 2, 90, 12
    st = dict(q=torch.zeros(4, Hq, D, dtype=torch.bfloat16, device="cuda"),
              lse=torch.zeros(4, Hq, device="cuda"), qs=gp.i32([0, 1, 4]), kv=gp.i32([200, 300]),
              tab=gp.i32([list(range(6)), list(range(6, 12))]))
    pages = gp.pool(911, num_pages, Hkv, True)
    w = torch.rand(num_pages, Hkv, PAGE, device="cuda")
    keep, n = gp.i32([[[0] * budget] * Hkv] * 2), gp.i32([0, 0])

    def evict():
        o.kv_weights(st["q"], st["lse"], pages, st["tab"], st["qs"], st["kv"], 3, 384, w, prev=w)
        o.kv_select(w, st["tab"], st["kv"], 384, budget, keep, n, sinks=4, recent=10)
        o.kv_keep(pages, st["tab"], keep, n, weights=w)

    state = [pages.k.view(torch.uint8), pages.vt.view(torch.uint8), pages.k_scale, pages.v_scale, w]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        evict()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        evict()
    g = torch.Generator().manual_seed(912)
    for lens in ([200, 300], [384, 64], [91, 89], [70, 384]):
        st["q"].copy_((torch.randn(4, Hq, D, generator=g) * gp.Q_SCALE).bfloat16())
        st["lse"].copy_(5 + torch.rand(4, Hq, generator=g))
        st["kv"].copy_(torch.tensor(lens, dtype=torch.int32))
        perm = torch.randperm(num_pages, generator=g).int()
        st["tab"].copy_(perm.view(2, 6))
        w.copy_(torch.rand(num_pages, Hkv, PAGE, generator=g))
        copy = [t.clone() for t in state]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*state, keep, n)]
        for t, old in zip(state, copy):
            t.copy_(old)
        evict()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (*state, keep, n)))


def test_pages_past_32_bits_of_a_pool():
    """Keys, weights and moves in pages whose offsets do not fit 32 bits."""
    o = gp.ops()
    Hkv, num_pages = 4, 35000  # 4.6 GB of K, 2^31 elements and more
    k = torch.zeros(num_pages, Hkv, PAGE, D, dtype=torch.bfloat16, device="cuda")
    vt = torch.zeros(num_pages, Hkv, D, PAGE, dtype=torch.bfloat16, device="cuda")
    pages = o.KvPages(k, vt)
    w = torch.zeros(num_pages, Hkv, PAGE, device="cuda")
    ids = [34999, 33000, 5, 34000]
    g = torch.Generator().manual_seed(921)
    k[ids] = torch.randn(4, Hkv, PAGE, D, generator=g).bfloat16().cuda()
    vt[ids] = torch.randn(4, Hkv, D, PAGE, generator=g).bfloat16().cuda()
    keep = sorted(random.Random(922).sample(range(192), 64))
    want_k = torch.stack([k[ids[p // PAGE], :, p % PAGE].clone() for p in keep], 1)
    want_v = torch.stack([vt[ids[p // PAGE], :, :, p % PAGE].clone() for p in keep], 2)
    q = (torch.randn(1, 4, D, generator=g) * gp.Q_SCALE).bfloat16()
    kc = k[ids[:3]].cpu().double().transpose(0, 1).reshape(Hkv, 192, D)
    o.kv_weights(q.cuda(), torch.zeros(1, 4, device="cuda"), pages, gp.i32([ids[:3]]),
                 gp.i32([0, 1]), gp.i32([192]), 1, 192, w)
    o.kv_keep(pages, gp.i32([ids[:3]]), gp.i32([[keep]]), gp.i32([64]),
              to_table=gp.i32([[34000]]), weights=w)
    torch.cuda.synchronize()
    ref = torch.exp2(torch.einsum("hd,hjd->hj", q[0].double(), kc))
    got = torch.cat([w[i].cpu().double() for i in ids[:3]], 1)
    assert ((got - ref).abs() <= 1e-4 * ref).all()
    assert torch.equal(k[34000], want_k) and torch.equal(vt[34000], want_v)
    assert torch.equal(w[34000], torch.cat([w[i] for i in ids[:3]], 1)[:, keep])
