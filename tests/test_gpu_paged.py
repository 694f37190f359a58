"""GPU tests of the paged K/V cache: writing new tokens into pages (bf16 and
e4m3), reading pages back, and attention over them, each against the float64
form in paged_oracle.py.

Tolerances: a rounding is off by at most half a step (bf16 2^-8 of the value,
e4m3 2^-4, or 2^-10 of the scale below its normal range); the fp32 arithmetic
before it adds 1e-5 of the row's largest magnitude (sums of 256 terms: 256 *
2^-24 = 1.5e-5 at the very most, of which the norm takes the root). V, scales of
V and everything read back are exact. The attention's bound is the oracle's.
"""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import paged_oracle as po  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D
EPS, ROT = 1e-6, 64
Q_SCALE = po.LOG2E / 16


def ops():
    from cujev import ops as o
    o.load()
    return o


def pool(seed, num_pages, Hkv, e4m3, garbage=False):
    """A pool whose slots all hold something: finite values as after other use,
    or (garbage) NaN in K, V and scales."""
    o = ops()
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(num_pages, Hkv, PAGE, D, generator=g).bfloat16()
    vt = torch.randn(num_pages, Hkv, D, PAGE, generator=g).bfloat16()
    if not e4m3:
        if garbage:
            k.fill_(math.nan), vt.fill_(math.nan)
        return o.KvPages(k.cuda(), vt.cuda())
    kq, ks = po.quantise(k.double(), 3)
    vq, vs = po.quantise(vt.double(), 2)
    kq, vq = kq.float().to(torch.float8_e4m3fn), vq.float().to(torch.float8_e4m3fn)
    ks, vs = ks.float(), vs.float()
    if garbage:
        kq.view(torch.uint8).fill_(0x7f), vq.view(torch.uint8).fill_(0x7f)
        ks.fill_(math.nan), vs.fill_(math.inf)
    return o.KvPages(kq.cuda(), vq.cuda(), ks.cuda(), vs.cuda())


def values(pages):
    """(K [np, Hkv, 64, D], V [np, Hkv, 64, D]) in float64 on the CPU."""
    k, v = pages.k.cpu().float().double(), pages.vt.cpu().float().double().transpose(2, 3)
    if pages.e4m3:
        k = k * pages.k_scale.cpu().double()[..., None]
        v = v * pages.v_scale.cpu().double()[..., None]
    return k, v


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def table(seed, kv_len, num_pages, max_pages=None):
    """Shuffled pages for each sequence; unused entries point nowhere."""
    ids = list(range(num_pages))
    random.Random(seed).shuffle(ids)
    need = [-(-max(k, 0) // PAGE) for k in kv_len]
    max_pages = max_pages or max(max(need), 1)
    out = []
    for n in need:
        out.append([ids.pop() for _ in range(n)] + [-1] * (max_pages - n))
    return out


def starts(q_lens):
    out = [0]
    for n in q_lens:
        out.append(out[-1] + n)
    return out


# ---- new tokens into pages ---------------------------------------------------
PREP = [
    # (Hq, Hkv, e4m3, [(new tokens, keys)])
    (8, 2, False, [(1, 1), (1, 64), (1, 65), (0, 10), (1, 130)]),
    (8, 2, True, [(1, 1), (1, 64), (1, 65), (0, 10), (1, 130)]),
    (16, 4, True, [(37, 37), (0, 0), (16, 80), (17, 97), (70, 200)]),
    (16, 4, False, [(37, 37), (0, 0), (16, 80), (17, 97), (70, 200)]),
    (4, 1, True, [(130, 131)]),
    (6, 1, True, [(5, 3), (64, 128), (3, 66)]),     # the first has fewer keys than tokens
    (16, 2, False, [(3, 66)] * 3 + [(0, 5)] * 70 + [(2, 63)] * 70),  # more than 64 sequences
    (4, 4, True, [(2, 63)] * 70 + [(33, 90)]),
    (4, 1, False, [(1, 3), (0, 5), (2, 66)] * 1500),  # past 64 x 64 of them
]


@pytest.mark.parametrize("Hq,Hkv,e4m3,lens", PREP)
def test_prep_writes_pages(Hq, Hkv, e4m3, lens):
    o = ops()
    q_lens, kv_len = [n for n, _ in lens], [k for _, k in lens]
    qs, N, extra = starts(q_lens), sum(q_lens), 3  # rows behind the last sequence
    num_pages = sum(-(-k // PAGE) for k in kv_len) + 2
    pages = pool(1, num_pages, Hkv, e4m3)
    tab = table(2, kv_len, num_pages)
    g = torch.Generator().manual_seed(3)
    width = Hq * 512 + Hkv * 512
    proj = torch.randn(N + extra, width + 8, generator=g).bfloat16()
    proj[:, Hq * 512 + Hkv * 256:] *= torch.exp2(torch.randint(-9, 9, (N + extra, 1), generator=g))
    if N > 2:
        proj[1, Hq * 512 + Hkv * 256:] = 0  # a V row of zeros
    qw, kw = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    pos = torch.randint(0, 500, (N + extra,), generator=g, dtype=torch.int32)
    rope = o.rope_table(1e7, ROT, 500)
    q_out = torch.full((N + extra, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    before = [t.clone() for t in (pages.k, pages.vt)]
    o.attn_prep_paged(proj.cuda()[:, :width + 8], qw.cuda(), kw.cuda(), pos.cuda(), i32(qs),
                      i32(kv_len), i32(tab), Hq, ROT, rope, EPS, Q_SCALE, q_out, pages)
    torch.cuda.synchronize()
    cs = rope.cpu().double()[pos.long()][:, None]
    x = proj.double()
    q = po.norm_rope(x[:, :Hq * 512].view(-1, Hq, 512)[..., :D], qw.double(), cs[..., 0],
                     cs[..., 1], ROT, EPS) * Q_SCALE
    k = po.norm_rope(x[:, Hq * 512:Hq * 512 + Hkv * 256].view(-1, Hkv, D), kw.double(),
                     cs[..., 0], cs[..., 1], ROT, EPS)
    v = x[:, Hq * 512 + Hkv * 256:width].view(-1, Hkv, D)
    got = q_out.cpu().double()
    assert ((got - q)[:N].abs() <= q[:N].abs() * 2 ** -8 +
            1e-5 * q[:N].abs().amax(-1, keepdim=True)).all()
    assert (got[N:] == 7.0).all(), "rows behind the last sequence were written"
    gk, gv = pages.k.cpu().float().double(), pages.vt.cpu().float().double()
    written = torch.zeros(num_pages, PAGE, dtype=torch.bool)
    for b in range(len(kv_len)):
        for n, _, page, slot in po.slots(qs, kv_len, tab, b, num_pages):
            written[page, slot] = True
            if e4m3:
                sk, sv = pages.k_scale[page, :, slot].cpu().double(), \
                    pages.v_scale[page, :, slot].cpu().double()
                vq, vs = po.quantise(v[n], 1)
                assert torch.equal(sv, vs), (b, n)
                assert torch.equal(gv[page, :, :, slot], vq), (b, n)
                a = k[n].abs().amax(1)
                assert (a <= 448 * sk * (1 + 1e-5)).all() and (a > 223.99 * sk).all()
                bound = k[n].abs() * 2 ** -4 + sk[:, None] * 2 ** -10 + 1e-5 * a[:, None]
                assert ((gk[page, :, slot] * sk[:, None] - k[n]).abs() <= bound).all(), (b, n)
            else:
                assert torch.equal(gv[page, :, :, slot], v[n]), (b, n)
                bound = k[n].abs() * 2 ** -8 + 1e-5 * k[n].abs().amax(1, keepdim=True)
                assert ((gk[page, :, slot] - k[n]).abs() <= bound).all(), (b, n)
    keep = ~written[:, None, :, None].cuda()
    as_bytes = (lambda t: t.view(torch.uint8)) if e4m3 else (lambda t: t)
    same = as_bytes(pages.k) == as_bytes(before[0])
    assert (same | ~keep).all(), "a K slot of no new token changed"
    same = as_bytes(pages.vt) == as_bytes(before[1])
    assert (same | ~keep.transpose(2, 3)).all(), "a V slot of no new token changed"


def test_prep_rounds_e4m3_keys_once():
    """K of e4m3 pages is the 64-bit value rounded once: every byte and scale of
    4 million values, some of tokens of zeros and of tiny and large ones."""
    o = ops()
    Hq, Hkv, N = 4, 4, 4000
    g = torch.Generator().manual_seed(181)
    width = Hq * 512 + Hkv * 512
    proj = torch.randn(N, width, generator=g).bfloat16()
    proj[7] = 0
    proj[8:12] *= torch.tensor([1e-3, 1e-12, 1e4, 1e12])[:, None].bfloat16()
    kw = 1 + 0.1 * torch.randn(D, generator=g)
    pos = torch.randint(0, 500, (N,), generator=g, dtype=torch.int32)
    rope = o.rope_table(1e7, ROT, 500)
    pages, tab = pool(182, 64, Hkv, True), table(183, [N], 64)
    q_out = torch.empty(N, Hq, D, dtype=torch.bfloat16, device="cuda")
    o.attn_prep_paged(proj.cuda(), kw.cuda(), kw.cuda(), pos.cuda(), i32([0, N]), i32([N]),
                      i32(tab), Hq, ROT, rope, EPS, Q_SCALE, q_out, pages)
    torch.cuda.synchronize()
    cs = rope.cpu().double()[pos.long()][:, None]
    k = po.norm_rope(proj.double()[:, Hq * 512:Hq * 512 + Hkv * 256].view(-1, Hkv, D), kw.double(),
                     cs[..., 0], cs[..., 1], ROT, EPS)
    kq, ks = po.quantise(k, 2)
    at = torch.tensor(tab[0])[:-(-N // PAGE)]
    gk = pages.k.cpu().float().double()[at].transpose(1, 2).reshape(-1, Hkv, D)[:N]
    gs = pages.k_scale.cpu().double()[at].transpose(1, 2).reshape(-1, Hkv)[:N]
    assert torch.equal(gs, ks)
    assert torch.equal(gk, kq)


def test_prep_skips_pages_that_are_not_there():
    """Ids outside the pool, lengths past the table: nothing is written there."""
    o = ops()
    pages = pool(1, 4, 2, True)
    before = [t.clone() for t in (pages.k, pages.vt, pages.k_scale, pages.v_scale)]
    N, Hq = 10, 8
    proj = torch.randn(N, Hq * 512 + 2 * 512, device="cuda").bfloat16()
    w = torch.ones(D, device="cuda")
    q_out = torch.empty(N, Hq, D, dtype=torch.bfloat16, device="cuda")
    rope = o.rope_table(1e7, ROT, 4)
    # ids 4 and -1; 200 keys of a table of 128; positions past the RoPE table and below 0
    o.attn_prep_paged(proj, w, w, i32([5, -3, 2, 1, 0, 9, 9, 9, 9, 9]), i32([0, 4, 8, 10]),
                      i32([66, 200, 1]), i32([[4, -1], [0, 1], [2 ** 30, 3]]), Hq, ROT, rope, EPS,
                      Q_SCALE, q_out, pages)
    torch.cuda.synchronize()
    for a, b in zip(before, (pages.k, pages.vt, pages.k_scale, pages.v_scale)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.isfinite(q_out.float()).all()


def test_prep_keeps_nan_and_infinity_to_their_rows():
    """A NaN or infinity becomes NaN in its own element; V rows beside it are exact."""
    o = ops()
    Hq, N = 4, 16
    pages = o.kv_pages(1, 1, e4m3=True)
    g = torch.Generator().manual_seed(5)
    proj = torch.randn(N, Hq * 512 + 512, generator=g).bfloat16()
    at = Hq * 512 + 256
    proj[3, at + 7], proj[9, at + 200] = math.nan, -math.inf
    w = torch.ones(D, device="cuda")
    q_out = torch.empty(N, Hq, D, dtype=torch.bfloat16, device="cuda")
    o.attn_prep_paged(proj.cuda(), w, w, i32(list(range(N))), i32([0, N]), i32([N]), i32([[0]]),
                      Hq, ROT, o.rope_table(1e7, ROT, N), EPS, Q_SCALE, q_out, pages)
    torch.cuda.synchronize()
    got = pages.vt.float().cpu()[0, 0]
    bad = torch.zeros(D, PAGE, dtype=torch.bool)
    bad[7, 3] = bad[200, 9] = True
    assert torch.equal(torch.isnan(got), bad)
    for t in (0, 2, 4, 8, 10, 15):
        vq, vs = po.quantise(proj[t, at:].double(), 0)
        assert torch.equal(got[:, t].double(), vq)
        assert pages.v_scale[0, 0, t].item() == vs.item()


# ---- pages back into caches ------------------------------------------------------
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hkv,kv_len", [(4, [530]), (2, [1, 64, 0, 65, 200]), (1, [63, 129])])
def test_read_gives_the_stored_values(Hkv, kv_len, e4m3):
    o = ops()
    num_pages = sum(-(-k // PAGE) for k in kv_len) + 1
    pages = pool(11, num_pages, Hkv, e4m3)
    tab = table(12, kv_len, num_pages)
    max_kv = max(kv_len)
    st = o.kv_stride(max_kv) + 64
    kc = torch.full((len(kv_len), Hkv, st, D), 5.0, dtype=torch.bfloat16, device="cuda")
    vc = torch.full((len(kv_len), Hkv, D, st), 5.0, dtype=torch.bfloat16, device="cuda")
    o.kv_page_read(pages, i32(tab), i32(kv_len), max_kv, kc, vc)
    torch.cuda.synchronize()
    k, v = values(pages)
    want_k, want_v = torch.full_like(kc.cpu(), 5.0).double(), torch.full_like(vc.cpu(), 5.0).double()
    for b, n in enumerate(kv_len):
        for p in range(n):
            want_k[b, :, p] = k[tab[b][p // PAGE], :, p % PAGE]
            want_v[b, :, :, p] = v[tab[b][p // PAGE], :, p % PAGE]
    assert torch.equal(kc.cpu().double(), want_k)
    assert torch.equal(vc.cpu().double(), want_v)


def test_read_of_missing_pages_is_zero_and_cut_to_max_kv():
    o = ops()
    pages = pool(13, 3, 1, True, garbage=True)
    kc = torch.full((1, 1, 256, D), 5.0, dtype=torch.bfloat16, device="cuda")
    vc = torch.full((1, 1, D, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    o.kv_page_read(pages, i32([[-1, 3, 2 ** 31 - 1]]), i32([10 ** 9]), 130, kc, vc)
    torch.cuda.synchronize()
    assert (kc[:, :, :130] == 0).all() and (kc[:, :, 130:] == 5).all()
    assert (vc[..., :130] == 0).all() and (vc[..., 130:] == 5).all()


# ---- attention ---------------------------------------------------------------------
def attention_case(seed, Hq, Hkv, e4m3, lens, extra=2, share=False):
    q_lens, kv_len = [n for n, _ in lens], [k for _, k in lens]
    num_pages = sum(-(-max(k, 0) // PAGE) for k in kv_len) + 3
    pages = pool(seed, num_pages, Hkv, e4m3)
    tab = table(seed + 1, kv_len, num_pages)
    if share:  # every sequence has the first one's first page as its own first
        for row, k in zip(tab, kv_len):
            if k > 0:
                row[0] = tab[0][0]
    g = torch.Generator().manual_seed(seed + 2)
    N = sum(q_lens) + extra
    q = (torch.randn(N, Hq, D, generator=g) * Q_SCALE).bfloat16()
    gate = torch.randn(N, Hq, D, generator=g).bfloat16()
    return dict(pages=pages, tab=tab, q=q, gate=gate, qs=starts(q_lens), kv_len=kv_len, N=N, Hq=Hq,
                Hkv=Hkv, e4m3=e4m3, max_q=max(q_lens), max_kv=max(max(kv_len), 0))


def run_attention(c, window=0, sinks=0, gate=True, max_q=None, max_kv=None):
    o = ops()
    max_q, max_kv = max_q or c["max_q"], max_kv or c["max_kv"]
    N, Hq = c["N"], c["Hq"]
    qg = torch.zeros(N, Hq, 2 * D, dtype=torch.bfloat16, device="cuda")
    qg[..., D:] = c["gate"].cuda()
    out = torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    nb = o.attention_paged_ws_bytes(N, len(c["kv_len"]), max_q, max_kv, Hq, c["Hkv"], window,
                                    sinks, c["e4m3"])
    # a workspace that holds NaN: nothing in it may be read before it is written
    ws = torch.full((nb // 4,), math.nan, device="cuda").view(torch.uint8) if nb else None
    o.attention_paged(c["q"].cuda(), qg[..., D:] if gate else None, Hq * 2 * D, 2 * D, c["pages"],
                      i32(c["tab"]), i32(c["qs"]), i32(c["kv_len"]), max_q, max_kv, out,
                      window=window, sinks=sinks, ws=ws)
    torch.cuda.synchronize()
    return out.cpu().double().view(N, Hq, D)


def check_attention(c, window=0, sinks=0, gate=True, **kw):
    got = run_attention(c, window, sinks, gate, **kw)
    k, v = values(c["pages"])
    K, V, there = [], [], []
    for b, n in enumerate(c["kv_len"]):
        at = [c["tab"][b][p // PAGE] for p in range(n)]
        there.append(torch.tensor([0 <= a < k.shape[0] for a in at], dtype=torch.bool))
        at = [a if 0 <= a < k.shape[0] else 0 for a in at]
        at, slot = torch.tensor(at, dtype=torch.long), torch.arange(max(n, 0)) % PAGE
        K.append(k[at, :, slot].transpose(0, 1))
        V.append(v[at, :, slot].transpose(0, 1))
    ref, tol = po.attention(c["q"].double(), c["gate"].double() if gate else None, K, V, there,
                            c["qs"], c["kv_len"], window, sinks)
    rows = c["qs"][-1]
    assert (got[rows:] == 7.0).all(), "rows behind the last sequence were written"
    assert torch.isfinite(got[:rows]).all()
    over = (got - ref)[:rows].abs() - tol[:rows]
    assert (over <= 0).all(), f"off by {over.max():.3g} over the bound, at {int(over.argmax())}"
    return got


ATTN = [
    # (Hq, Hkv, [(new tokens, keys)], window, sinks)
    (8, 2, [(1, 1)], 0, 0),
    (8, 2, [(1, 530)], 0, 0),
    (16, 4, [(1, 1), (1, 64), (1, 65), (1, 127), (1, 300), (0, 70), (1, 128)], 0, 0),
    (4, 1, [(1, 1500), (1, 20)], 0, 0),
    (6, 1, [(1, 200), (1, 77)], 0, 0),
    (16, 1, [(1, 200), (1, 77)], 0, 0),
    (4, 4, [(1, 200), (1, 77)], 0, 0),
    (8, 2, [(4, 300), (3, 90), (1, 5)], 0, 0),          # a few tokens each
    (8, 2, [(8, 300), (5, 90), (1, 5), (0, 0)], 0, 0),
    (8, 2, [(40, 300), (1, 90), (33, 33)], 0, 0),
    (16, 4, [(64, 64), (65, 200)], 0, 0),
    (4, 1, [(150, 700)], 0, 0),
    (6, 1, [(50, 130), (21, 21), (43, 100)], 0, 0),
    (3, 3, [(140, 200)], 0, 0),
    (8, 2, [(5, 3), (1, 0), (2, 2)], 0, 0),             # rows before position 0: no keys
    (8, 2, [(1, 1), (1, 530), (1, 129)], 64, 0),        # windows
    (8, 2, [(1, 1), (1, 530), (1, 129)], 64, 4),
    (8, 2, [(1, 900), (1, 700)], 100, 70),              # sinks past a tile
    (8, 2, [(1, 200)], 1, 0),                           # a token sees itself alone
    (8, 2, [(1, 200), (3, 130)], 1, 1),
    (16, 4, [(100, 400), (64, 64), (1, 300)], 50, 3),
    (4, 1, [(200, 600)], 128, 64),
    (4, 1, [(90, 300)], 1000, 10),                      # a window past the start
    (4, 1, [(90, 300)], 7, 500),                        # sinks past the window
    (6, 1, [(70, 200)], 33, 5),
]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens,window,sinks", ATTN)
def test_attention_matches_oracle(Hq, Hkv, lens, window, sinks, e4m3):
    print(f"case Hq={Hq} Hkv={Hkv} lens={lens} window={window} sinks={sinks} e4m3={e4m3}",
          flush=True)
    check_attention(attention_case(21, Hq, Hkv, e4m3, lens), window, sinks)


@pytest.mark.parametrize("e4m3", [False, True])
def test_attention_without_gate_and_with_loose_bounds(e4m3):
    """No gate; max_q and max_kv far above the lengths give the same rows."""
    c = attention_case(31, 8, 2, e4m3, [(3, 70), (1, 260)])
    check_attention(c, gate=False)
    c["tab"] = [row + [-1] * 40 for row in c["tab"]]
    check_attention(c, gate=False, max_q=3, max_kv=2000)
    check_attention(c, gate=False, max_q=200, max_kv=2000)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("q", [1, 30])
def test_attention_of_more_than_64_sequences(q, e4m3):
    r = random.Random(7)
    lens = [(r.choice([0, 1, q]), r.randint(q, 90)) for _ in range(150)]
    lens[3] = (q, 90)
    check_attention(attention_case(41, 4, 1, e4m3, lens, share=True))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(1, 400), (1, 90)], [(40, 400), (3, 70)]])
def test_attention_skips_pages_that_are_not_there(lens, e4m3):
    """A page id outside the pool hides its keys; a row left with none gives 0."""
    c = attention_case(51, 8, 2, e4m3, lens)
    c["tab"][0][1], c["tab"][0][3] = -1, 2 ** 30
    check_attention(c)
    c["tab"][1] = [-5] * len(c["tab"][1])
    got = check_attention(c)
    assert (got[c["qs"][1]:c["qs"][2]] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,window,sinks", [
    ([(1, 100), (1, 64), (1, 65)], 0, 0), ([(1, 500), (1, 150)], 80, 3),
    ([(50, 100), (64, 64), (1, 70)], 0, 0), ([(40, 500), (30, 170)], 80, 3),
])
def test_attention_ignores_what_no_row_sees(lens, window, sinks, e4m3):
    """NaN in every slot that no row of the call sees (behind the last key, before
    the window, in other pages, in the scales) changes nothing."""
    c = attention_case(61, 8, 2, e4m3, lens)
    clean = check_attention(c, window, sinks)
    dirty = pool(61, c["pages"].num_pages, 2, e4m3, garbage=True)
    for b, (n, kv) in enumerate(lens):
        for p in range(kv):
            lo = kv - n - window + 1 if window else 0
            if p < lo and p >= sinks:
                continue
            page, slot = c["tab"][b][p // PAGE], p % PAGE
            dirty.k[page, :, slot] = c["pages"].k[page, :, slot]
            dirty.vt.view(torch.uint8 if e4m3 else torch.bfloat16)[page, :, :, slot] = \
                c["pages"].vt.view(torch.uint8 if e4m3 else torch.bfloat16)[page, :, :, slot]
            if e4m3:
                dirty.k_scale[page, :, slot] = c["pages"].k_scale[page, :, slot]
                dirty.v_scale[page, :, slot] = c["pages"].v_scale[page, :, slot]
    c["pages"] = dirty
    assert torch.equal(run_attention(c, window, sinks), clean)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(1, 300), (1, 70)], [(40, 300), (3, 70)]])
@pytest.mark.parametrize("scale", [900.0, -900.0, 30.0])
def test_attention_of_large_scores(lens, scale, e4m3):
    """Scores of thousands either way: the softmax's reference moves."""
    c = attention_case(71, 8, 2, e4m3, lens)
    k = c["pages"].k
    if e4m3:
        c["pages"].k_scale.mul_(64.0)
    else:
        k.mul_(64.0)
    c["q"] = (c["q"].float().abs() * scale / 64).bfloat16()  # all scores lean one way
    if e4m3:
        k.view(torch.uint8).bitwise_and_(0x7f)
    else:
        k.abs_()
    got = run_attention(c)
    kk, v = values(c["pages"])
    for b, (n, kv) in enumerate(lens):
        for i in range(n):
            row, p = c["qs"][b] + i, kv - n + i
            at = [c["tab"][b][j // PAGE] for j in range(p + 1)]
            slot = torch.arange(p + 1) % PAGE
            for h in range(8):
                K, V = kk[at, h // 4, slot], v[at, h // 4, slot]
                x = K @ c["q"][row, h].double()
                # what an error of the fp32 scores can do, each way
                es = 256 * 2.0 ** -24 * 2 * (K.abs() @ c["q"][row, h].double().abs())
                pr = torch.exp2(x - x.max())
                pr /= pr.sum()
                o = (pr @ V) * torch.sigmoid(c["gate"][row, h].double())
                spread = ((pr * (torch.exp2(es + es.max()) - 1)) @ (V.abs() + V.abs().max()))
                tol = spread + (pr @ V.abs() + o.abs()) * 2.0 ** -8 * 1.01 + 1e-6
                assert ((got[row, h] - o).abs() <= tol).all(), (b, i, h)


# ---- together ------------------------------------------------------------------------
def test_a_sequence_through_pages_is_the_same_as_through_a_state():
    """Prompt of 150, then 3 single tokens, by attn_prep + attention on contiguous
    caches and by the paged operators on bf16 pages: the same q and K / V bits,
    outputs within both kernels' roundings; read back, the state's caches."""
    o = ops()
    Hq, Hkv, T = 16, 4, 153
    g = torch.Generator().manual_seed(81)
    proj = torch.randn(T, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    qw, kw = (1 + 0.1 * torch.randn(D, generator=g)).cuda(), (1 + 0.1 * torch.randn(D, generator=g)).cuda()
    rope = o.rope_table(1e7, ROT, 256)
    pos = i32(list(range(T)))
    st = o.kv_stride(T)
    kc = torch.zeros(Hkv, st, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros(Hkv, D, st, dtype=torch.bfloat16, device="cuda")
    q1 = torch.empty(T, Hq, D, dtype=torch.bfloat16, device="cuda")
    o.attn_prep(proj, qw, kw, pos, Hq, Hkv, ROT, rope, EPS, Q_SCALE, q1, kc, vc, st)
    out1 = torch.empty(T, Hq * D, dtype=torch.bfloat16, device="cuda")
    gate = proj[:, D:]
    o.attention(q1, gate, proj.stride(0), 512, kc, vc, 0, st, kc, vc, st,
                torch.zeros(T, dtype=torch.int32, device="cuda"), Hq, Hkv, out1)
    pages = o.kv_pages(5, Hkv)
    tab = i32([[3, 0, 4]])
    q2, out2 = torch.empty_like(q1), torch.empty_like(out1)
    for n0, n1 in ((0, 150), (150, 151), (151, 152), (152, 153)):
        qs, kv = i32([0, n1 - n0]), i32([n1])
        o.attn_prep_paged(proj[n0:n1], qw, kw, pos[n0:n1], qs, kv, tab, Hq, ROT, rope, EPS,
                          Q_SCALE, q2[n0:n1], pages)
        nb = o.attention_paged_ws_bytes(n1 - n0, 1, n1 - n0, n1, Hq, Hkv)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None
        o.attention_paged(q2[n0:n1], gate[n0:n1], proj.stride(0), 512, pages, tab, qs, kv, n1 - n0,
                          n1, out2[n0:n1], ws=ws)
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    o.kv_page_read(pages, tab, i32([T]), T, kc2[None], vc2[None])
    torch.cuda.synchronize()
    assert torch.equal(q1, q2) and torch.equal(kc, kc2) and torch.equal(vc, vc2)
    # each is within 2^-8 (p) and 2^-8 (output) of the exact result: |v| averages
    # out to at most the largest |v| a row sees
    a, b = out1.float(), out2.float()
    lim = vc.float().abs().max()
    assert ((a - b).abs() <= 2 * 2 ** -8 * (lim + a.abs())).all()
    assert ((a - b).norm() / a.norm()).item() < 4 * 2 ** -9


def test_a_parked_state_answers_branches_after_it_is_read_back():
    """prep into e4m3 pages -> kv_page_read -> cujev_op_attention of branches over
    the restored state: what attention_paged gives for the same branch as new
    tokens of the sequence."""
    o = ops()
    Hq, Hkv, P, L = 8, 2, 200, 20
    g = torch.Generator().manual_seed(91)
    proj = torch.randn(P + L, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    w = torch.ones(D, device="cuda")
    rope, pos = o.rope_table(1e7, ROT, 512), i32(list(range(P + L)))
    pages, tab = o.kv_pages(6, Hkv, e4m3=True), i32([[5, 1, 2, 0]])
    q = torch.empty(P + L, Hq, D, dtype=torch.bfloat16, device="cuda")
    for n0, n1 in ((0, P), (P, P + L)):
        o.attn_prep_paged(proj[n0:n1], w, w, pos[n0:n1], i32([0, n1 - n0]), i32([n1]), tab, Hq,
                          ROT, rope, EPS, Q_SCALE, q[n0:n1], pages)
    st = o.kv_stride(P + L)
    kc = torch.zeros(Hkv, st, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros(Hkv, D, st, dtype=torch.bfloat16, device="cuda")
    o.kv_page_read(pages, tab, i32([P + L]), P + L, kc[None], vc[None])
    # the branch's own keys, as the branch scratch holds them
    ost = o.kv_stride(L)
    ok = torch.zeros(Hkv, ost, D, dtype=torch.bfloat16, device="cuda")
    ovt = torch.zeros(Hkv, D, ost, dtype=torch.bfloat16, device="cuda")
    ok[:, :L], ovt[..., :L] = kc[:, P:P + L], vc[..., P:P + L]
    gate = proj[P:, D:]
    out1 = torch.empty(L, Hq * D, dtype=torch.bfloat16, device="cuda")
    o.attention(q[P:], gate, proj.stride(0), 512, kc, vc, P, st, ok, ovt, ost,
                torch.zeros(L, dtype=torch.int32, device="cuda"), Hq, Hkv, out1)
    out2 = torch.empty_like(out1)
    nb = o.attention_paged_ws_bytes(L, 1, L, P + L, Hq, Hkv, e4m3=True)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None
    o.attention_paged(q[P:], gate, proj.stride(0), 512, pages, tab, i32([0, L]), i32([P + L]), L,
                      P + L, out2, ws=ws)
    torch.cuda.synchronize()
    a, b = out1.float(), out2.float()
    assert ((a - b).abs() <= 2 * 2 ** -8 * (vc.float().abs().max() + a.abs())).all()


def test_a_captured_step_replays_with_other_lengths_and_tables():
    """prep + attention of one token per sequence captured once, replayed as the
    sequences grow: every replay equals the eager calls."""
    o = ops()
    Hq, Hkv, B, steps, max_kv = 8, 2, 5, 6, 200
    g = torch.Generator().manual_seed(101)
    proj = torch.randn(steps, B, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    w, rope = torch.ones(D, device="cuda"), o.rope_table(1e7, ROT, 256)
    tab, qs = i32(table(102, [max_kv] * B, 25)), i32(list(range(B + 1)))
    lens = [[60, 63, 64, 100, 0], [61, 64, 65, 101, 1], [62, 65, 66, 180, 2], [63, 66, 67, 181, 3],
            [64, 67, 68, 182, 4], [65, 68, 69, 190, 5]]
    nb = o.attention_paged_ws_bytes(B, B, 1, max_kv, Hq, Hkv, e4m3=True)

    def state():
        return dict(pages=pool(103, 25, Hkv, True), kv=i32([1] * B), pos=i32([0] * B),
                    proj=torch.empty_like(proj[0]),
                    q=torch.empty(B, Hq, D, dtype=torch.bfloat16, device="cuda"),
                    out=torch.empty(B, Hq * D, dtype=torch.bfloat16, device="cuda"),
                    ws=torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None)

    def step(s):
        o.attn_prep_paged(s["proj"], w, w, s["pos"], qs, s["kv"], tab, Hq, ROT, rope, EPS,
                          Q_SCALE, s["q"], s["pages"])
        o.attention_paged(s["q"], s["proj"][:, D:], s["proj"].stride(0), 512, s["pages"], tab, qs,
                          s["kv"], 1, max_kv, s["out"], ws=s["ws"])

    a, b = state(), state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for i in range(steps):
        for s in (a, b):
            s["proj"].copy_(proj[i])
            s["kv"].copy_(i32(lens[i]))
            s["pos"].copy_((i32(lens[i]) - 1).clamp(min=0))
        step(a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a["out"], b["out"]), i
        assert torch.equal(a["pages"].vt.view(torch.uint8), b["pages"].vt.view(torch.uint8)), i
        assert torch.equal(a["pages"].k.view(torch.uint8), b["pages"].k.view(torch.uint8)), i


def test_calls_run_on_the_current_stream_and_repeat_bit_for_bit():
    o = ops()
    c = attention_case(111, 16, 4, True, [(1, 900), (1, 64), (1, 333)])
    first = run_attention(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = run_attention(c)
    assert torch.equal(first, again)


def _lens_over_pieces(seed):
    """Sequences of every length up to 11 pages, and many in a row without a token."""
    g = torch.Generator().manual_seed(seed)
    kv = torch.randint(1, 700, (150,), generator=g).tolist()
    return [(0 if 20 <= i < 100 or i % 7 == 3 else 1, k) for i, k in enumerate(kv)]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_attention_of_one_token_over_many_uneven_sequences(window, sinks, e4m3):
    c = attention_case(121, 16, 4, e4m3, _lens_over_pieces(122))
    check_attention(c, window, sinks)
    # of bounds far above the lengths, the work is shared out otherwise
    check_attention(c, window, sinks, max_q=3, max_kv=700)


@pytest.mark.parametrize("q", [1, 40])
def test_attention_of_hundreds_of_sequences(q):
    """More than the 256 that a step of the plan takes, with and without shares."""
    g = torch.Generator().manual_seed(191)
    lens = [(min(int(n), q), int(k)) for n, k in zip(torch.randint(0, q + 1, (700,), generator=g),
                                                     torch.randint(40, 150, (700,), generator=g))]
    check_attention(attention_case(192, 4, 1, False, lens), max_kv=150)
    lens = [(0, 9)] * 600 + [(q, 1400), (1, 70)] + [(0, 9)] * 100
    check_attention(attention_case(193, 4, 1, True, lens))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,lens", [
    (4, [(0, 0)] * 15 + [(1, 9000)]),  # one sequence has all of the work of 16
    (16, [(1, 9000)]),
    (4, [(33, 17000)]),                # units of more than 16 shares
    (4, [(1400, 1400), (60, 90)]),     # a new sequence: its first units stay whole
    (1, [(130, 2500), (1, 3)]),
])
def test_attention_in_many_parts(Hq, lens, e4m3):
    check_attention(attention_case(131, Hq, 1, e4m3, lens))


@pytest.mark.parametrize("Hq,Hkv", [(5, 1), (10, 2), (7, 1), (13, 1), (22, 2), (15, 1)])
@pytest.mark.parametrize("lens", [[(1, 300), (1, 64)], [(30, 300), (11, 11)]])
def test_attention_of_odd_head_groups(Hq, Hkv, lens):
    check_attention(attention_case(141, Hq, Hkv, True, lens))


def test_calls_on_two_streams_at_once():
    """Calls with workspaces of their own, in flight together, give what each
    gives alone."""
    o = ops()
    cases = [attention_case(151, 16, 4, True, [(1, 3000)] * 6),
             attention_case(152, 8, 2, False, [(40, 2000), (3, 700)])]
    alone = [run_attention(c) for c in cases]
    calls, streams = [], [torch.cuda.Stream() for _ in cases]
    for c in cases:
        N, Hq = c["N"], c["Hq"]
        qg = torch.zeros(N, Hq, 2 * D, dtype=torch.bfloat16, device="cuda")
        qg[..., D:] = c["gate"].cuda()
        nb = o.attention_paged_ws_bytes(N, len(c["kv_len"]), c["max_q"], c["max_kv"], Hq, c["Hkv"],
                                        e4m3=c["e4m3"])
        assert nb > 0
        outs = [torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
                for _ in range(8)]
        calls.append((c["q"].cuda(), qg[..., D:], Hq * 2 * D, 2 * D, c["pages"], i32(c["tab"]),
                      i32(c["qs"]), i32(c["kv_len"]), c["max_q"], c["max_kv"], outs,
                      torch.empty(nb, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for i in range(8):
        for s, a in zip(streams, calls):
            with torch.cuda.stream(s):
                o.attention_paged(*a[:-2], a[-2][i], ws=a[-1])
    torch.cuda.synchronize()
    for a, ref, c in zip(calls, alone, cases):
        for out in a[-2]:
            assert torch.equal(out.cpu().double().view(c["N"], c["Hq"], D), ref)


def test_a_captured_prefill_replays_with_other_lengths():
    """prep + attention of many tokens a sequence, in shares that are merged:
    every replay equals the eager calls, rows of no sequence stay."""
    o = ops()
    Hq, Hkv, B, N, max_q, max_kv = 8, 2, 3, 90, 40, 2600
    g = torch.Generator().manual_seed(161)
    width = Hq * 512 + Hkv * 512
    w, rope = torch.ones(D, device="cuda"), o.rope_table(1e7, ROT, max_kv)
    tab = i32(table(162, [max_kv] * B, 130))
    steps = [([40, 40, 10], [2600, 40, 1000]), ([1, 0, 40], [2000, 0, 64]),
             ([40, 30, 20], [40, 2599, 2600]), ([0, 0, 1], [0, 5, 1])]
    nb = o.attention_paged_ws_bytes(N, B, max_q, max_kv, Hq, Hkv)
    assert nb > 0

    def state():
        return dict(pages=pool(163, 130, Hkv, False), kv=i32([1] * B), pos=i32([0] * N),
                    qs=i32([0] * (B + 1)),
                    proj=torch.zeros(N, width, dtype=torch.bfloat16, device="cuda"),
                    q=torch.zeros(N, Hq, D, dtype=torch.bfloat16, device="cuda"),
                    out=torch.zeros(N, Hq * D, dtype=torch.bfloat16, device="cuda"),
                    ws=torch.empty(nb, dtype=torch.uint8, device="cuda"))

    def step(s):
        o.attn_prep_paged(s["proj"], w, w, s["pos"], s["qs"], s["kv"], tab, Hq, ROT, rope, EPS,
                          Q_SCALE, s["q"], s["pages"])
        o.attention_paged(s["q"], s["proj"][:, D:], width, 512, s["pages"], tab, s["qs"], s["kv"],
                          max_q, max_kv, s["out"], ws=s["ws"])

    a, b = state(), state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for q_lens, kv in steps:
        proj = torch.randn(N, width, generator=g).bfloat16().cuda()
        pos = [p for n, k in zip(q_lens, kv) for p in range(k - n, k)]
        for s in (a, b):
            s["proj"].copy_(proj)
            s["kv"].copy_(i32(kv))
            s["qs"].copy_(i32(starts(q_lens)))
            s["pos"].copy_(i32(pos + [0] * (N - len(pos))))
            s["out"].fill_(7.0)
        step(a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a["out"], b["out"]), q_lens
        assert torch.equal(a["pages"].k, b["pages"].k) and torch.equal(a["pages"].vt, b["pages"].vt)
        assert (a["out"][sum(q_lens):] == 7.0).all()


def test_pages_past_32_bits_of_a_pool():
    """The last pages of a pool of more than 2^32 bytes (and 2^31 values) give
    what the same pages give in a small one."""
    o = ops()
    Hq, Hkv, lens, n = 8, 8, [(1, 300), (20, 150), (1, 64)], 16600
    c = attention_case(171, Hq, Hkv, False, lens)
    used = c["pages"].num_pages
    big = o.KvPages(torch.empty(n, Hkv, PAGE, D, dtype=torch.bfloat16, device="cuda"),
                    torch.empty(n, Hkv, D, PAGE, dtype=torch.bfloat16, device="cuda"))
    assert big.k.numel() > 2 ** 31
    big.k[n - used:].copy_(c["pages"].k)
    big.vt[n - used:].copy_(c["pages"].vt)
    high = [[p + n - used for p in row] for row in c["tab"]]
    N = c["qs"][-1]
    proj = torch.randn(N, Hq * 512 + Hkv * 512, device="cuda").bfloat16()
    w, rope = torch.ones(D, device="cuda"), o.rope_table(1e7, ROT, 512)
    pos = i32([p for q, k in lens for p in range(k - q, k)])
    got = []
    for pages, tab in ((c["pages"], c["tab"]), (big, high)):
        q = torch.empty(N, Hq, D, dtype=torch.bfloat16, device="cuda")
        out = torch.empty(N, Hq * D, dtype=torch.bfloat16, device="cuda")
        kc, vc = (torch.zeros(s, dtype=torch.bfloat16, device="cuda")
                  for s in ((3, Hkv, o.kv_stride(300), D), (3, Hkv, D, o.kv_stride(300))))
        nb = o.attention_paged_ws_bytes(N, 3, 20, 300, Hq, Hkv)
        ws = torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None
        t, qs, kv = i32(tab), i32(c["qs"]), i32(c["kv_len"])
        o.attn_prep_paged(proj, w, w, pos, qs, kv, t, Hq, ROT, rope, EPS, Q_SCALE, q, pages)
        o.attention_paged(q, None, 0, 0, pages, t, qs, kv, 20, 300, out, ws=ws)
        o.kv_page_read(pages, t, kv, 300, kc, vc)
        got.append((q, out, kc, vc))
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a, b)
