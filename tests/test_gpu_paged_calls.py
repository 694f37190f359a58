"""GPU tests of the paged K/V cache's calls as a server makes them: one workspace
for all, and lengths, strides and values at the ends of their ranges. Inputs,
oracle and tolerances are test_gpu_paged.py's and paged_oracle.py's.
"""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_oracle as po  # noqa: E402
import test_gpu_paged as gp  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D


def oracle(c, window=0, sinks=0, gate=True, there=None):
    """(out, tolerance) of the case; `there`: per sequence the keys that are there."""
    k, v = gp.values(c["pages"])
    K, V, keys = [], [], []
    for b, n in enumerate(c["kv_len"]):
        at = [c["tab"][b][p // PAGE] for p in range(n)]
        at, slot = torch.tensor(at, dtype=torch.long), torch.arange(n) % PAGE
        K.append(k[at, :, slot].transpose(0, 1))
        V.append(v[at, :, slot].transpose(0, 1))
        keys.append(torch.ones(n, dtype=torch.bool) if there is None else there[b])
    return po.attention(c["q"].double(), c["gate"].double() if gate else None, K, V, keys,
                        c["qs"], c["kv_len"], window, sinks)


def run(c, ws, window=0, sinks=0, gate=True, max_q=None, max_kv=None):
    """attention_paged with this workspace, checked against nothing."""
    o, N, Hq = gp.ops(), c["N"], c["Hq"]
    g = c["gate"].cuda() if gate else None
    out = torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    o.attention_paged(c["q"].cuda(), g, Hq * D, D, c["pages"], gp.i32(c["tab"]), gp.i32(c["qs"]),
                      gp.i32(c["kv_len"]), c["max_q"] if max_q is None else max_q,
                      c["max_kv"] if max_kv is None else max_kv, out, window=window, sinks=sinks,
                      ws=ws)
    torch.cuda.synchronize()
    return out.cpu().double().view(N, Hq, D)


def check(got, ref, tol, rows):
    assert torch.isfinite(got[:rows]).all()
    over = (got - ref)[:rows].abs() - tol[:rows]
    assert (over <= 0).all(), f"off by {over.max():.3g} over the bound, at {int(over.argmax())}"


def test_one_workspace_serves_a_prompt_and_the_steps_after_it():
    """Sized for a call of 2200 new tokens, whose rows fill the chip: chunks, single
    tokens, windows and both types of pages go through it, full of NaN before each."""
    Hq, Hkv = 16, 4
    nb = gp.ops().attention_paged_ws_bytes(2200, 3, 2200, 2200, Hq, Hkv)
    assert nb > 0
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    for i, (lens, window, sinks, e4m3) in enumerate([
            ([(2200, 2200)], 0, 0, False), ([(40, 2200), (20, 900)], 0, 0, False),
            ([(40, 2200), (20, 900)], 0, 0, True), ([(1, 2200), (1, 300), (1, 64)], 0, 0, True),
            ([(1, 2200), (1, 300)], 1000, 4, False), ([(60, 2200)], 1500, 4, True)]):
        print(f"case {lens} window={window} sinks={sinks} e4m3={e4m3}", flush=True)
        c = gp.attention_case(201 + 3 * i, Hq, Hkv, e4m3, lens)
        ws.view(torch.float32).fill_(math.nan)
        got = run(c, ws, window, sinks)
        if i == 0:  # every 100th row: the oracle goes row by row
            k, v = gp.values(c["pages"])
            at, slot = torch.tensor(c["tab"][0])[torch.arange(2200) // PAGE], torch.arange(2200) % PAGE
            K, V = k[at, :, slot].transpose(0, 1), v[at, :, slot].transpose(0, 1)
            for n in range(0, 2200, 100):
                ref, tol = po.attention(c["q"][n:n + 1].double(), c["gate"][n:n + 1].double(),
                                        [K[:, :n + 1]], [V[:, :n + 1]],
                                        [torch.ones(n + 1, dtype=torch.bool)], [0, 1], [n + 1], 0,
                                        0)
                check(got[n:n + 1], ref, tol, 1)
            continue
        check(got, *oracle(c, window, sinks), c["qs"][-1])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(1, 400), (3, 130), (1, 90)], [(50, 400), (20, 90)]])
@pytest.mark.parametrize("window,sinks", [(128, 0), (128, 4), (150, 0), (200, 70), (1000, 4),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
def test_rows_past_max_kv_keep_their_window(window, sinks, lens, e4m3):
    """Sequences of more than max_kv = 128 keys with a window of at least that: a row
    sees the keys before max_kv that its window or the sinks hold, and no others."""
    o = gp.ops()
    c = gp.attention_case(231, 8, 2, e4m3, lens)
    nb = o.attention_paged_ws_bytes(c["N"], len(lens), c["max_q"], 128, 8, 2)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None
    there = [torch.arange(kv) < 128 for _, kv in lens]
    got = run(c, ws, window, sinks, max_kv=128)
    check(got, *oracle(c, window, sinks, there=there), c["qs"][-1])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,max_q", [([(8, 300), (2, 90), (5, 64)], 3),
                                        ([(60, 300), (20, 90), (70, 70)], 25)])
def test_tokens_past_max_q_reach_no_row(lens, max_q, e4m3):
    """Of a sequence of more than max_q new tokens the first max_q are computed, the
    others' rows stay as they were, and their keys, NaN here, are none of the call's."""
    o, nan = gp.ops(), math.nan
    c = gp.attention_case(241, 8, 2, e4m3, lens)
    ref, tol = oracle(c)
    pages = c["pages"]
    for b, (n, kv) in enumerate(lens):
        for p in range(kv - n + min(n, max_q), kv):
            page, slot = c["tab"][b][p // PAGE], p % PAGE
            for t in (pages.k[page, :, slot], pages.vt[page, :, :, slot]):
                t.view(torch.uint8).fill_(0x7f) if e4m3 else t.fill_(nan)
            if e4m3:
                pages.k_scale[page, :, slot], pages.v_scale[page, :, slot] = nan, nan
    nb = o.attention_paged_ws_bytes(c["N"], len(lens), max_q, c["max_kv"], 8, 2)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda") if nb else None
    got = run(c, ws, max_q=max_q)
    for b, (n, kv) in enumerate(lens):
        q0, q1, q2 = c["qs"][b], c["qs"][b] + min(n, max_q), c["qs"][b + 1]
        check(got[q0:q1], ref[q0:q1], tol[q0:q1], q1 - q0)
        assert (got[q1:q2] == 7.0).all(), "a row past max_q was written"


@pytest.mark.parametrize("e4m3", [False, True])
def test_read_of_negative_lengths_writes_nothing(e4m3):
    """Down to the least int, whose distance to a page's first key is none."""
    o = gp.ops()
    pages = gp.pool(251, 5, 1, e4m3)
    kv_len = [-2 ** 31, -1, -2 ** 31 + 100, 3, -64]
    kc = torch.full((5, 1, 256, D), 5.0, dtype=torch.bfloat16, device="cuda")
    vc = torch.full((5, 1, D, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    o.kv_page_read(pages, gp.i32([[0, 1, 2, 3]] * 5), gp.i32(kv_len), 190, kc, vc)
    torch.cuda.synchronize()
    k, v = gp.values(pages)
    want_k, want_v = torch.full(kc.shape, 5.0).double(), torch.full(vc.shape, 5.0).double()
    want_k[3, :, :3], want_v[3, :, :, :3] = k[0, :, :3], v[0, :, :3].transpose(1, 2)
    assert torch.equal(kc.cpu().double(), want_k) and torch.equal(vc.cpu().double(), want_v)


def uneven(seed, B, lo, hi, most):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(lo, hi + 1, (B,), generator=g).tolist()
    return [(n, n + int(torch.randint(0, most, (1,), generator=g))) for n in q]


# (Hq, Hkv, [(new tokens, keys)]): V by groups with a wave a page, which takes more than
# 1024 waves' worth of groups at fewer than 128 rows a sequence; by rows; a wave a group
BY_PAGES = [(16, 4, uneven(261, 50, 5, 50, 250)), (8, 4, uneven(262, 64, 40, 64, 70)),
            (4, 4, uneven(263, 40, 0, 90, 30)), (16, 8, uneven(264, 30, 17, 100, 500)),
            (16, 4, [(5, 3), (0, 0), (40, 20)] + uneven(265, 60, 10, 40, 64))]
BY_ROWS = [(8, 2, uneven(266, 80, 0, 3, 200))]
BY_GROUPS = [(16, 4, uneven(267, 5, 1, 70, 200)), (4, 1, [(130, 131), (1, 64)])]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", BY_PAGES)
def test_prep_of_chunks_of_many_sequences(Hq, Hkv, lens, e4m3):
    N, B = sum(n for n, _ in lens) + 3, len(lens)  # three rows behind the last
    assert min(N, N // PAGE + 2 * B) * Hkv * 4 > 1024 and N < 128 * B and not (B > 64 and N <= 3 * B)
    gp.test_prep_writes_pages(Hq, Hkv, e4m3, lens)


@pytest.mark.parametrize("Hq,Hkv,lens", BY_PAGES + BY_ROWS + BY_GROUPS)
def test_prep_leaves_the_scales_of_other_slots(Hq, Hkv, lens):
    """Every byte of the pool that no new token has, scales among them, stays; a page id
    outside the pool leaves all of its tokens' out."""
    o = gp.ops()
    q_lens, kv_len = [n for n, _ in lens], [k for _, k in lens]
    qs, N = gp.starts(q_lens), sum(q_lens)
    num_pages = sum(-(-k // PAGE) for k in kv_len) + 2
    pages, tab = gp.pool(271, num_pages, Hkv, True), gp.table(272, kv_len, num_pages)
    tab[0][0], tab[-1][-1] = -1, num_pages
    for t in (pages.k, pages.vt, pages.k_scale, pages.v_scale):  # no value that prep writes
        t.view(torch.uint8).fill_(0x7f)
    g = torch.Generator().manual_seed(273)
    proj = torch.randn(N, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    w = torch.ones(D, device="cuda")
    q_out = torch.empty(N, Hq, D, dtype=torch.bfloat16, device="cuda")
    o.attn_prep_paged(proj, w, w, gp.i32([0] * N), gp.i32(qs), gp.i32(kv_len), gp.i32(tab), Hq,
                      gp.ROT, o.rope_table(1e7, gp.ROT, 4), gp.EPS, gp.Q_SCALE, q_out, pages)
    torch.cuda.synchronize()
    written = torch.zeros(num_pages, PAGE, dtype=torch.bool)
    for b in range(len(kv_len)):
        for _, _, page, slot in po.slots(qs, kv_len, tab, b, num_pages):
            written[page, slot] = True
    written = written[:, None, :].expand(-1, Hkv, -1)
    same = lambda t, dim: (t.cpu().view(torch.uint8) == 0x7f).all(dim)
    for name, t in (("k_scale", pages.k_scale), ("v_scale", pages.v_scale)):
        kept = same(t.reshape(num_pages, Hkv, PAGE, 1), 3)
        assert torch.equal(kept, ~written), name
    assert torch.equal(same(pages.k, 3), ~written)
    assert torch.equal(same(pages.vt, 2), ~written)


@pytest.mark.parametrize("e4m3", [False, True])
def test_prep_of_one_row_of_any_stride(e4m3):
    """A single row's stride says nothing: a column turned over gives a row's bits."""
    o = gp.ops()
    Hq, Hkv = 4, 1
    g = torch.Generator().manual_seed(281)
    row = torch.randn(1, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    w, rope = torch.ones(D, device="cuda"), o.rope_table(1e7, gp.ROT, 4)
    column = row.reshape(-1, 1).clone().t()
    assert column.stride(0) == 1
    got = []
    for proj in (row, column, row.as_strided(row.shape, (2 ** 33, 1))):
        pages = o.kv_pages(1, Hkv, e4m3)
        q = torch.empty(1, Hq, D, dtype=torch.bfloat16, device="cuda")
        o.attn_prep_paged(proj, w, w, gp.i32([3]), gp.i32([0, 1]), gp.i32([4]), gp.i32([[0]]), Hq,
                          gp.ROT, rope, gp.EPS, gp.Q_SCALE, q, pages)
        got.append((q, pages.k, pages.vt))
    torch.cuda.synchronize()
    assert got[0][0].any()
    for other in got[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got[0], other))


SCORES = {
    # the score of (row n of N, key j of kv), up to noise
    "62": lambda n, N, j, kv: 62.0, "-62": lambda n, N, j, kv: -62.0,
    "30": lambda n, N, j, kv: 30.0, "-30": lambda n, N, j, kv: -30.0,
    "by row": lambda n, N, j, kv: -62.0 + 124.0 * n / max(N - 1, 1),
    "rising": lambda n, N, j, kv: 62.0 * (2 * j / kv - 1), "far": lambda n, N, j, kv: 400.0,
}


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(1, 300), (3, 64), (2, 1500)], [(40, 1500), (33, 90), (1, 70)]])
@pytest.mark.parametrize("size", [80, 40, 0, -40, -64])
@pytest.mark.parametrize("scores", list(SCORES))
def test_values_of_any_magnitude_and_scores_together(scores, size, lens, e4m3):
    """V of up to 2^80 and down to 2^-64 beside scores of up to 62 either way, where the
    softmax's reference may stay 0 and p comes to 2^62 or 2^-62."""
    o = gp.ops()
    Hq, Hkv = 8, 2
    c = gp.attention_case(291, Hq, Hkv, False, lens)
    g = torch.Generator().manual_seed(292)
    shape = c["pages"].k.shape
    score, N = SCORES[scores], c["qs"][-1]
    by_key = scores == "rising"
    k = 1 + 0.05 * torch.randn(shape, generator=g)
    if by_key:
        for b, (_, kv) in enumerate(lens):
            for j in range(kv):
                k[c["tab"][b][j // PAGE], :, j % PAGE] *= score(0, N, j, kv) / 62
    vt = (2 * torch.rand(c["pages"].vt.shape, generator=g) - 1) * 2.0 ** size
    for n in range(N):
        c["q"][n] = (62.0 if by_key else score(n, N, 0, 1)) / 256
    if e4m3:
        kq, ks = po.quantise(k.double(), 3)
        vq, vs = po.quantise(vt.double(), 2)
        f8 = lambda t: t.float().to(torch.float8_e4m3fn).cuda()
        c["pages"] = o.KvPages(f8(kq), f8(vq), ks.float().cuda(), vs.float().cuda())
    else:
        c["pages"] = o.KvPages(k.bfloat16().cuda(), vt.bfloat16().cuda())
    nb = o.attention_paged_ws_bytes(c["N"], len(lens), c["max_q"], c["max_kv"], Hq, Hkv)
    got = run(c, torch.empty(nb, dtype=torch.uint8, device="cuda"))
    ref, tol = oracle(c)
    check(got, ref, tol, N)
    assert (got[N:] == 7.0).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_single_tokens_beside_a_prompt(window, sinks, e4m3):
    """A step of 63 sequences with one more's prompt in it: one call, of tiles of many
    rows for all."""
    g = torch.Generator().manual_seed(301)
    lens = [(1, int(k)) for k in torch.randint(1, 1500, (63,), generator=g)]
    lens.insert(20, (200, 900))
    c = gp.attention_case(302, 8, 2, e4m3, lens)
    gp.check_attention(c, window, sinks)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(3, 300), (2, 64)], [(40, 300), (33, 90)]])
def test_rows_before_the_first_sequence_and_no_keys_at_all(lens, e4m3):
    """q_start may begin behind row 0; with max_kv 0 no row sees a key; with max_q 0 no
    row is one of the call's."""
    o = gp.ops()
    c = gp.attention_case(311, 8, 2, e4m3, lens)
    ref, tol = oracle(c)
    nb = o.attention_paged_ws_bytes(c["N"] + 5, 2, c["max_q"], c["max_kv"], 8, 2)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    pad = lambda t: torch.cat([torch.full_like(t[:5], math.nan), t])
    late = {**c, "q": pad(c["q"]), "gate": pad(c["gate"]), "N": c["N"] + 5,
            "qs": [n + 5 for n in c["qs"]]}
    got, rows = run(late, ws), c["qs"][-1]
    assert (got[:5] == 7.0).all() and (got[5 + rows:] == 7.0).all()
    check(got[5:], ref, tol, rows)
    got = run(c, ws, max_kv=0)
    assert (got[:rows] == 0.0).all() and (got[rows:] == 7.0).all()
    assert (run(c, ws, max_q=0) == 7.0).all()
    # prep: the same rows, K and V from row 5 on
    Hq, Hkv, N = 8, 2, c["N"] + 5
    g = torch.Generator().manual_seed(312)
    proj = torch.randn(N, Hq * 512 + Hkv * 512, generator=g).bfloat16().cuda()
    w, rope = torch.ones(D, device="cuda"), o.rope_table(1e7, gp.ROT, 4)
    outs = []
    for first, at in ((5, gp.i32(late["qs"])), (0, gp.i32(c["qs"]))):
        pages = o.kv_pages(c["pages"].num_pages, Hkv, e4m3)
        q = torch.full((N - 5 + first, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
        o.attn_prep_paged(proj[5 - first:], w, w, gp.i32([1] * (N - 5 + first)), at,
                          gp.i32(c["kv_len"]), gp.i32(c["tab"]), Hq, gp.ROT, rope, gp.EPS,
                          gp.Q_SCALE, q, pages)
        outs.append((q[first:], pages.k, pages.vt))
        assert (q[:first] == 7.0).all() and (q[first + rows:] == 7.0).all()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*outs))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens,bad", [([(3, 300), (2, 64)], [1]), ([(40, 1500), (33, 90)], [5, 50])])
def test_a_row_of_nan_or_infinity_stays_a_row(lens, bad, e4m3):
    """q that is not finite in a row (and a head) reaches no other."""
    c = gp.attention_case(321, 8, 2, e4m3, lens)
    ref, tol = oracle(c)
    c["q"][bad[0], 3], c["q"][bad[-1], 5, 7] = math.nan, math.inf
    nb = gp.ops().attention_paged_ws_bytes(c["N"], 2, c["max_q"], c["max_kv"], 8, 2)
    got, rows = run(c, torch.empty(nb, dtype=torch.uint8, device="cuda")), c["qs"][-1]
    for n, h in ((bad[0], 3), (bad[-1], 5)):
        got[n, h], ref[n, h], tol[n, h] = 0.0, 0.0, 0.0
    check(got, ref, tol, rows)


@pytest.mark.parametrize("e4m3", [False, True])
def test_single_tokens_and_prompts_in_a_call_each(e4m3):
    """One batch in two calls over parts of q_start, kv_len and page_table: each writes its
    own sequences' rows, and both together the whole batch's."""
    o = gp.ops()
    n, lens = 5, [(1, 900), (1, 64), (1, 1), (0, 30), (1, 333), (60, 700), (90, 90), (0, 0)]
    c = gp.attention_case(331, 8, 2, e4m3, lens)
    nb = o.attention_paged_ws_bytes(c["N"], len(lens), c["max_q"], c["max_kv"], 8, 2)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    q, gate = c["q"].cuda(), c["gate"].cuda()
    tab, qs, kv = gp.i32(c["tab"]), gp.i32(c["qs"]), gp.i32(c["kv_len"])
    out = torch.full((c["N"], 8 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    for seqs, starts, max_q in ((slice(0, n), slice(0, n + 1), 1),
                                (slice(n, None), slice(n, None), c["max_q"])):
        o.attention_paged(q, gate, 8 * D, D, c["pages"], tab[seqs], qs[starts], kv[seqs], max_q,
                          c["max_kv"], out, ws=ws)
        if max_q == 1:
            torch.cuda.synchronize()
            assert (out[c["qs"][n]:] == 7.0).all()
    torch.cuda.synchronize()
    got, rows = out.cpu().double().view(-1, 8, D), c["qs"][-1]
    check(got, *oracle(c), rows)
    assert (got[rows:] == 7.0).all()
