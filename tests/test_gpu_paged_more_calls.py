"""GPU tests of how draft trees, attention weights and eviction may be called: two calls
at once, sequences that share pages, a budget of nothing."""
import pytest

torch = pytest.importorskip("torch")

import evict_oracle as eo  # noqa: E402
import paged_oracle as po  # noqa: E402
import test_gpu_evict as ge  # noqa: E402
import test_gpu_paged as gp  # noqa: E402
import test_gpu_paged_tree as gt  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D


def on_device(c, tree):
    """A call's tensors and a workspace of its own, and the call."""
    o = gp.ops()
    N, Hq = c["N"], c["Hq"]
    q, g, lse = c["q"].cuda(), c["gate"].cuda(), c["lse"].cuda()
    tab, qs, kv = gp.i32(c["tab"]), gp.i32(c["qs"]), gp.i32(c["kv_len"])
    nb = o.attention_paged_ws_bytes(N, len(c["kv_len"]), c["max_q"], c["max_kv"], Hq, c["Hkv"])
    wb = o.kv_weights_ws_bytes(N, len(c["kv_len"]), c["max_q"], c["max_kv"], Hq, c["Hkv"])
    ws = torch.empty(max(nb, wb, 16), dtype=torch.uint8, device="cuda")
    t = tree.cuda()

    def call():
        out = torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
        got, w = torch.full((N, Hq), 7.0, device="cuda"), c["w"].cuda()
        o.attention_paged(q, g, Hq * D, D, c["pages"], tab, qs, kv, c["max_q"], c["max_kv"], out,
                          ws=ws, tree=t, lse=got)
        o.kv_weights(q, lse, c["pages"], tab, qs, kv, c["max_q"], c["max_kv"], w, prev=w, ws=ws)
        return out, got, w
    return call


@pytest.mark.parametrize("e4m3", [False, True])
def test_two_calls_at_once(e4m3):
    """On two streams, each with a workspace of its own that its calls share in turn."""
    calls = []
    for seed, lens in ((401, [(12, 900), (9, 400)]), (402, [(40, 3000), (33, 97)])):
        c = gt.tree_case(seed, 16, 4, e4m3, lens)
        calls.append(on_device(ge.fill(c, seed), c["tree"]))
    torch.cuda.synchronize()
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = calls[i]()
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(want[i], got[i]):
            # bit for bit: rows of no sequence hold 7, pages of none what they held
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(4, 260), (3, 200)], [(20, 600), (13, 540)]])
def test_trees_of_sequences_that_share_a_prefix(lens, e4m3):
    """Whole pages before the new tokens belong to both sequences."""
    c = gt.tree_case(411, 8, 2, e4m3, lens)
    shared = min(kv - n for n, kv in lens) // PAGE
    assert shared > 1
    c["tab"][1][:shared] = c["tab"][0][:shared]
    got, lse = gt.run(c, c["tree"])
    gt.check(c, got, lse, gt.tree_seen(c))


def test_a_budget_of_nothing():
    o = gp.ops()
    w = torch.rand(4, 2, PAGE).cuda()
    keep = torch.empty(2, 2, 0, dtype=torch.int32, device="cuda")
    keep_len = gp.i32([9, 9])
    o.kv_select(w, gp.i32([[0, 1], [2, 3]]), gp.i32([100, 0]), 128, 0, keep, keep_len)
    assert keep_len.tolist() == [0, 0]


@pytest.mark.parametrize("e4m3", [False, True])
def test_weights_of_a_draft_by_its_accepted_rows(e4m3):
    """A draft's accepted tokens, moved to lie in a row: their rows' q and lse of the tree
    give the weights that causal attention over what is kept gives them."""
    o, lens = gp.ops(), [(26, 530), (12, 200)]
    c = gt.tree_case(421, 16, 4, e4m3, lens)
    _, lse = gt.run(c, c["tree"])
    paths = []
    for b, (n, _) in enumerate(lens):
        deep = max(range(n), key=lambda i: int(c["seen"][b][i].sum()))
        paths.append(c["seen"][b][deep].nonzero()[:, 0].tolist())
    most = max(map(len, paths))
    keep = torch.tensor([[[kv - n + i for i in (p + [0] * most)[:most]]]
                         for p, (n, kv) in zip(paths, lens)], dtype=torch.int32)
    before = [kv - n for n, kv in lens]
    o.kv_keep(c["pages"], gp.i32(c["tab"]), keep.cuda(), gp.i32([len(p) for p in paths]),
              dst=gp.i32(before))
    torch.cuda.synchronize()
    rows = [c["qs"][b] + i for b, p in enumerate(paths) for i in p]
    a = {**c, "q": c["q"][rows], "N": len(rows), "max_q": most,
         "qs": [0, len(paths[0]), len(rows)],
         "kv_len": [at + len(p) for at, p in zip(before, paths)]}
    a["lse"] = lse[rows].float()
    shape = (c["pages"].num_pages, 4, PAGE)
    g = torch.Generator().manual_seed(5)
    a["prev"], a["w"] = torch.rand(*shape, generator=g), torch.rand(*shape, generator=g)
    ge.check_weights(a, ge.weigh(a))
    # and the lse of the tree is that of causal rows
    for b in range(2):
        q0, ql, p0, kv = eo.rows_of(a, b)
        K, _, _ = gt.cache(a, b, kv)
        seen = gt.causal()(b, p0, ql, kv)
        for h in range(16):
            want, tol, _ = eo.attend(a["q"][q0:q0 + ql, h].double(), K[h // 4], seen)
            assert ((a["lse"][q0:q0 + ql, h].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("slope", [0.02, 0.05, 0.2, -0.2])
@pytest.mark.parametrize("lens", [[(4, 700), (2, 64)], [(13, 700), (9, 64), (16, 300)],
                                  [(40, 700), (33, 97)]])
def test_trees_of_scores_that_rise_from_key_to_key(lens, slope, e4m3):
    """By more or less a tile than moves the softmax's reference."""
    c = gt.tree_case(431, 16, 4, e4m3, lens)
    k = torch.zeros(c["pages"].k.shape)
    for b, (_, kv) in enumerate(lens):
        for p in range(kv):
            k[c["tab"][b][p // PAGE], :, p % PAGE, 0] = slope * p
    c["pages"].k.copy_(k.to(c["pages"].k.dtype))
    if e4m3:
        c["pages"].k_scale.fill_(1.0)
    c["q"][..., 0] = 1.0
    got, lse = gt.run(c, c["tree"])
    gt.check(c, got, lse, gt.tree_seen(c))


def test_captured_weights_of_a_prompt_replay_with_other_lengths():
    """Rows shared out among workgroups, the workspace from torch's allocator in the graph."""
    o = gp.ops()
    Hq, Hkv, num_pages, most = 8, 2, 24, 400
    pages = gp.pool(441, num_pages, Hkv, False)
    st = dict(q=torch.zeros(most, Hq, D, dtype=torch.bfloat16, device="cuda"),
              lse=torch.zeros(most, Hq, device="cuda"), qs=gp.i32([0, 200, 400]),
              kv=gp.i32([200, 300]), tab=gp.i32([list(range(12)), list(range(12, 24))]))
    w = torch.rand(num_pages, Hkv, PAGE, device="cuda")
    assert o.kv_weights_ws_bytes(most, 2, 300, 768, Hq, Hkv) > 0

    def weigh():
        o.kv_weights(st["q"], st["lse"], pages, st["tab"], st["qs"], st["kv"], 300, 768, w, prev=w)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        weigh()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        weigh()
    g = torch.Generator().manual_seed(442)
    for qs, lens in (([0, 200, 400], [200, 768]), ([0, 1, 290], [700, 289]),
                     ([0, 300, 300], [768, 5]), ([0, 130, 400], [129, 500])):
        st["q"].copy_((torch.randn(most, Hq, D, generator=g) * gp.Q_SCALE).bfloat16())
        st["lse"].copy_(5 + torch.rand(most, Hq, generator=g))
        st["qs"].copy_(torch.tensor(qs, dtype=torch.int32))
        st["kv"].copy_(torch.tensor(lens, dtype=torch.int32))
        st["tab"].copy_(torch.randperm(num_pages, generator=g).int().view(2, 12))
        before = torch.rand(num_pages, Hkv, PAGE, generator=g)
        w.copy_(before)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = w.clone()
        w.copy_(before)
        weigh()
        torch.cuda.synchronize()
        assert torch.equal(got, w)


@pytest.mark.parametrize("lens", [[(3, 190)], [(13, 190)], [(70, 190)]])
def test_trees_in_pages_past_32_bits_of_a_pool(lens):
    """The bits of the same pages at the front of a small pool."""
    o = gp.ops()
    c = gt.tree_case(451, 16, 4, False, lens)
    want, want_lse = gt.run(c, c["tree"])
    num_pages, ids = 35000, [34999, 33000, 34000]  # 4.6 GB of K, 2^31 elements and more
    k = torch.zeros(num_pages, 4, PAGE, D, dtype=torch.bfloat16, device="cuda")
    vt = torch.zeros(num_pages, 4, D, PAGE, dtype=torch.bfloat16, device="cuda")
    k[ids], vt[ids] = c["pages"].k[c["tab"][0][:3]], c["pages"].vt[c["tab"][0][:3]]
    got, lse = gt.run({**c, "pages": o.KvPages(k, vt), "tab": [ids]}, c["tree"])
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
