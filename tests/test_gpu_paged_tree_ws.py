"""GPU tests of draft trees in workspaces of every size, against the float64 forms of
evict_oracle.py."""
import math

import pytest

torch = pytest.importorskip("torch")

import paged_oracle as po  # noqa: E402
import test_gpu_paged as gp  # noqa: E402
import test_gpu_paged_tree as gt  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D
LENS = [[(26, 530)], [(8, 512)] * 5 + [(3, 100), (0, 9)], [(60, 800), (33, 97)]]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", LENS)
def test_a_tree_in_a_workspace_of_a_causal_call(lens, e4m3):
    """The library's own entry: less than the form of 64 rows takes gives the other form."""
    o, Hq, Hkv = gp.ops(), 16, 4
    c = gt.tree_case(541, Hq, Hkv, e4m3, lens)
    N, B = c["N"], len(lens)
    size = o.attention_paged_ws_bytes(N, B, c["max_q"], c["max_kv"], Hq, Hkv)
    assert size < o.attention_paged_ws_bytes(N, B, c["max_q"], c["max_kv"], Hq, Hkv, tree=True)
    # what lies behind the size that is told is not the call's
    ws = torch.full((size // 4 + 4096,), math.nan, device="cuda")
    q, g, tree = c["q"].cuda(), c["gate"].cuda(), c["tree"].cuda()
    qs, kv, tab = gp.i32(c["qs"]), gp.i32(c["kv_len"]), gp.i32(c["tab"])
    out = torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((N, Hq), 7.0, device="cuda")
    st = o.load().cujev_op_attention_paged_tree(
        q.data_ptr(), g.data_ptr(), Hq * D, D, *c["pages"].args, qs.data_ptr(), kv.data_ptr(),
        tab.data_ptr(), tab.shape[1], B, N, c["max_q"], c["max_kv"], Hq, Hkv, tree.data_ptr(),
        c["tree"].shape[1], out.data_ptr(), lse.data_ptr(), ws.data_ptr(), size,
        torch.cuda.current_stream().cuda_stream)
    assert st == 0
    torch.cuda.synchronize()
    gt.check(c, out.cpu().double().view(N, Hq, D), lse.cpu().double(), gt.tree_seen(c))
    assert torch.isnan(ws[size // 4:]).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", LENS)
def test_the_binding_takes_a_workspace_where_one_is_too_small(lens, e4m3):
    """The bits of the call with a tree's own, without one and with a causal call's."""
    o, Hq, Hkv = gp.ops(), 16, 4
    c = gt.tree_case(551, Hq, Hkv, e4m3, lens)
    N, B = c["N"], len(lens)
    sizes = [o.attention_paged_ws_bytes(N, B, c["max_q"], c["max_kv"], Hq, Hkv, tree=t)
             for t in (True, False)]
    q, g, tree = c["q"].cuda(), c["gate"].cuda(), c["tree"].cuda()
    qs, kv, tab = gp.i32(c["qs"]), gp.i32(c["kv_len"]), gp.i32(c["tab"])
    got = []
    for size in (*sizes, 0):
        out = torch.full((N, Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((N, Hq), 7.0, device="cuda")
        o.attention_paged(q, g, Hq * D, D, c["pages"], tab, qs, kv, c["max_q"], c["max_kv"], out,
                          ws=torch.empty(size, dtype=torch.uint8, device="cuda") if size else None,
                          tree=tree, lse=lse)
        got.append((out, lse))
    torch.cuda.synchronize()
    out, lse = got[0]
    gt.check(c, out.cpu().double().view(N, Hq, D), lse.cpu().double(), gt.tree_seen(c))
    for a, b in got[1:]:
        assert torch.equal(a, out) and torch.equal(b, lse)
