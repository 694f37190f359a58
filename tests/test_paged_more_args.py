"""Refusals of the paged cache's further entry points (rotary axes, statistics, draft
trees, eviction), on the CPU: every call here is turned away by the host's checks
before anything is launched. The base cases are test_paged_args.py's."""
import pytest

torch = pytest.importorskip("torch")

from cujev import ops  # noqa: E402
import test_paged_args as pa  # noqa: E402
from test_paged_args import CAPACITY, FAKE, INVALID, POOL  # noqa: E402


def insert(args, after, **new):
    out = {}
    for k, v in args.items():
        out[k] = v
        if k == after:
            out.update(new)
    return out


AXES, LSE, TREE = ("cujev_op_attn_prep_paged_axes", "cujev_op_attention_paged_lse",
                   "cujev_op_attention_paged_tree")
WEIGHTS, SELECT, KEEP = "cujev_op_kv_weights", "cujev_op_kv_select", "cujev_op_kv_keep"
attn = pa.BASE[pa.ATTN]
BASE = {
    AXES: insert(pa.BASE[pa.PREP], "pos", axes=3, axis_of=0b100100),
    LSE: insert(attn, "out", lse=FAKE),
    TREE: insert(insert({k: v for k, v in attn.items() if k not in ("window", "sinks")}, "Hkv",
                        tree=FAKE, tree_words=1), "out", lse=None),
    WEIGHTS: dict(q=FAKE, lse=FAKE, kv_type=1, k_pages=FAKE, k_scale=FAKE, num_pages=4,
                  q_start=FAKE, kv_len=FAKE, page_table=FAKE, max_pages=2, B=0, N=0, max_q=1,
                  max_kv=128, Hq=8, Hkv=2, prev=None, weights=FAKE, ws=None, ws_bytes=0,
                  stream=None),
    SELECT: dict(weights=FAKE, num_pages=4, Hkv=2, page_table=FAKE, max_pages=2, kv_len=FAKE, B=0,
                 max_kv=128, budget=64, sinks=4, recent=16, keep=FAKE, max_keep=64,
                 keep_len=FAKE + 64, stream=None),
    KEEP: dict(kv_type=1, k_pages=FAKE, vt_pages=FAKE, k_scale=FAKE, v_scale=FAKE, weights=None,
               num_pages=4, Hkv=2, page_table=FAKE, max_pages=2, to_table=None, to_pages=0, B=0,
               keep=FAKE, keep_heads=2, max_keep=64, dst=None, keep_len=FAKE, stream=None),
}


def call(name, **changes):
    args = dict(BASE[name])
    assert set(changes) <= set(args), changes
    args.update(changes)
    lib = ops.load()
    return getattr(lib, name)(*args.values()), lib.cujev_ops_last_error().decode()


def test_argument_order_is_the_headers():
    for name, args in BASE.items():
        assert len(args) == len(ops._SIGS[name]), name


@pytest.mark.parametrize("name", list(BASE))
def test_an_empty_call_does_nothing(name):
    assert call(name)[0] == 0


@pytest.mark.parametrize("name", list(BASE))
@pytest.mark.parametrize("bad", pa.BAD_POOL, ids=str)
def test_pool_and_table_are_checked(name, bad):
    here = BASE[name]
    bad = {{"kv_len": "keep_len"}.get(k, k) if name == KEEP else k: v for k, v in bad.items()}
    if not set(bad) <= set(here):
        pytest.skip("no such argument")
    st, msg = call(name, **bad)
    assert st == INVALID and name[9:] in msg


@pytest.mark.parametrize("bad", [
    dict(axes=0), dict(axes=5), dict(axes=2), dict(axis_of=0b11), dict(axis_of=3 << 62), dict(N=-1),
    dict(Hq=7), dict(rot=24), dict(npos=0), dict(proj_stride=5119), dict(q_out=FAKE + 4),
    dict(N=1, B=1, pos=None)], ids=str)
def test_prep_of_axes_refuses(bad):
    st, msg = call(AXES, **bad)
    assert st == INVALID and "attn_prep_paged_axes" in msg


def test_axes_of_frequencies_that_there_are_not_are_not_looked_at():
    assert call(AXES, rot=8, axes=1, axis_of=0xff00)[0] == 0


@pytest.mark.parametrize("bad", [
    dict(N=1, B=1, lse=None), dict(lse=FAKE + 2), dict(window=-1), dict(sinks=4), dict(max_kv=129),
    dict(q=FAKE + 8), dict(N=-1), dict(Hq=34)], ids=str)
def test_lse_refuses(bad):
    st, msg = call(LSE, **bad)
    assert st == INVALID and "attention_paged_lse" in msg


@pytest.mark.parametrize("bad", [
    dict(N=1, B=1, tree=None), dict(tree=FAKE + 4), dict(lse=FAKE + 2), dict(tree_words=0),
    dict(tree_words=-1), dict(N=65, max_q=65), dict(N=300, max_q=200, tree_words=3),
    dict(max_kv=129), dict(N=-1), dict(Hq=34), dict(gate=FAKE + 2)], ids=str)
def test_tree_refuses(bad):
    st, msg = call(TREE, **bad)
    assert st == INVALID and "attention_paged_tree" in msg


@pytest.mark.parametrize("name", [LSE, TREE])
def test_a_workspace_that_is_too_small_is_refused(name):
    st, msg = call(name, N=1, B=1, ws=FAKE, ws_bytes=16)
    assert st == CAPACITY and "workspace" in msg


@pytest.mark.parametrize("bad", [
    dict(N=-1), dict(max_q=-1), dict(max_kv=-1), dict(max_kv=129), dict(Hq=7), dict(Hq=34),
    dict(N=1, B=1, q=None), dict(N=1, B=1, lse=None), dict(N=1, B=1, q_start=None),
    dict(N=1, B=1, weights=None), dict(q=FAKE + 8), dict(lse=FAKE + 1), dict(prev=FAKE + 2),
    dict(weights=FAKE + 3), dict(B=1 << 26, N=1)], ids=str)
def test_weights_refuse(bad):
    st, msg = call(WEIGHTS, **bad)
    assert st == INVALID and "kv_weights" in msg


def test_weights_refuse_a_workspace_that_is_too_small():
    need = ops.kv_weights_ws_bytes(1000, 1, 1000, 128, 8, 2)
    assert need > 0 and ops.kv_weights_ws_bytes(1000, 1, 32, 128, 8, 2) == 0
    for ws, size in ((None, 0), (FAKE, need - 1), (FAKE + 2, need)):
        st, msg = call(WEIGHTS, N=1000, B=1, max_q=1000, ws=ws, ws_bytes=size)
        assert st == CAPACITY and "workspace" in msg


@pytest.mark.parametrize("bad", [
    dict(max_kv=-1), dict(max_kv=129), dict(budget=-1), dict(sinks=-1), dict(recent=-1),
    dict(sinks=40, recent=25), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1, budget=2 ** 31 - 1),
    dict(max_keep=63), dict(B=1, weights=None), dict(B=1, keep=None), dict(B=1, keep_len=None),
    dict(B=1, keep_len=FAKE), dict(B=1 << 25)], ids=str)
def test_select_refuses(bad):
    st, msg = call(SELECT, **bad)
    assert st == INVALID and "kv_select" in msg


@pytest.mark.parametrize("bad", [
    dict(keep_heads=3), dict(keep_heads=0), dict(max_keep=-1), dict(max_keep=(1 << 28) + 1),
    dict(to_table=FAKE), dict(to_table=FAKE, to_pages=-1), dict(to_table=FAKE, to_pages=1 << 23),
    dict(B=1, keep=None), dict(B=1 << 28)], ids=str)
def test_keep_refuses(bad):
    st, msg = call(KEEP, **bad)
    assert st == INVALID and "kv_keep" in msg


def test_rope_axes():
    a = ops.RopeAxes.from_sections([11, 11, 10], interleaved=True)
    assert a.axes == 3 and len(a.axis_of) == 32
    assert [a.axis_of.count(i) for i in range(3)] == [11, 11, 10]
    assert a.axis_of[:6] == (0, 1, 2, 0, 1, 2) and a.axis_of[30:] == (0, 1)
    assert a.packed == sum(x << 2 * i for i, x in enumerate(a.axis_of))
    assert ops.RopeAxes.from_sections([2, 1, 1]).axis_of == (0, 0, 1, 2)
    for bad in ([], [4], [-1], [0] * 33):
        with pytest.raises(ops.OpsError):
            ops.RopeAxes(bad)


def host_calls(e4m3=False):
    """Calls that are right but for the memory: all on the CPU."""
    t = torch.float8_e4m3fn if e4m3 else torch.bfloat16
    sc = [torch.ones(2, 1, 64) for _ in range(2 * e4m3)]
    pages = ops.KvPages(torch.zeros(2, 1, 64, 256).to(t), torch.zeros(2, 1, 256, 64).to(t), *sc)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    seqs = dict(kv_len=i32(1), page_table=i32(0)[None])
    q, w = bf(1, 4, 256), torch.ones(256)
    attn = dict(q=q, gate=None, gate_tok_stride=0, gate_head_stride=0, pages=pages,
                q_start=i32(0, 1), max_q=1, max_kv=1, out=bf(1, 1024), **seqs)
    return {
        AXES: (ops.attn_prep_paged, dict(
            proj=bf(1, 2560), q_norm_w=w, k_norm_w=w, pos=i32(0, 0)[:, None], q_start=i32(0, 1),
            Hq=4, rot=64, rope=torch.zeros(8, 32, 2), eps=1e-6, q_scale=0.1, q_out=q, pages=pages,
            axes=ops.RopeAxes([0, 1] * 16), **seqs)),
        LSE: (ops.attention_paged, dict(attn, lse=torch.zeros(1, 4))),
        TREE: (ops.attention_paged, dict(attn, tree=torch.ones(1, 1, dtype=torch.int64))),
        WEIGHTS: (ops.kv_weights, dict(q=q, lse=torch.zeros(1, 4), pages=pages, q_start=i32(0, 1),
                                       max_q=1, max_kv=1, weights=torch.zeros(2, 1, 64), **seqs)),
        SELECT: (ops.kv_select, dict(weights=torch.zeros(2, 1, 64), max_kv=1, budget=1,
                                     keep=i32(0)[None, None], keep_len=i32(0), **seqs)),
        KEEP: (ops.kv_keep, dict(pages=pages, page_table=i32(0)[None], keep=i32(0)[None, None],
                                 keep_len=i32(1))),
    }


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("name", list(BASE))
def test_bindings_refuse_tensors_in_host_memory(name, e4m3, monkeypatch):
    """The library is a stand-in: nothing can be launched."""
    reached = []

    class Library:
        def __getattr__(self, symbol):
            return lambda *args: reached.append(symbol) or 0

    monkeypatch.setattr(ops, "_lib", Library())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0, raising=False)
    f, kw = host_calls(e4m3)[name]
    with pytest.raises(ops.OpsError, match="host memory"):
        f(**kw)
    assert not reached


def test_bindings_refuse_wrong_tensors():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    z = torch.zeros
    for name, bads in {
        AXES: [dict(pos=i32(0)), dict(pos=z(3, 1, dtype=torch.int32)),
               dict(axes=ops.RopeAxes([0, 1])), dict(pos=z(2, 1)), dict(axes=None)],
        LSE: [dict(lse=z(1, 3)), dict(lse=z(1, 4).double()), dict(lse=z(4))],
        TREE: [dict(tree=z(1, 1)), dict(tree=z(2, 1, dtype=torch.int64)),
               dict(tree=z(1, dtype=torch.int64)), dict(window=8), dict(window=8, sinks=2)],
        WEIGHTS: [dict(lse=z(1, 3)), dict(lse=None), dict(q=z(1, 4, 256)), dict(q=z(4, 256)),
                  dict(weights=z(2, 1, 63)), dict(weights=z(1, 1, 64)), dict(weights=None),
                  dict(prev=z(2, 1, 64).double()), dict(max_kv=2 ** 32), dict(max_q=-1),
                  dict(kv_len=i32(1, 1)), dict(q_start=i32(0)), dict(ws=z(8))],
        SELECT: [dict(weights=z(2, 1, 32)), dict(weights=z(2, 64)), dict(weights=z(2, 1, 64).double()),
                 dict(keep=i32(0)), dict(keep=z(1, 2, 1, dtype=torch.int32)),
                 dict(keep_len=i32(0, 0)), dict(kv_len=torch.tensor([1])), dict(page_table=i32(0)),
                 dict(budget=2 ** 31), dict(sinks=-1)],
        KEEP: [dict(keep=i32(0)), dict(keep=z(1, 2, 1, dtype=torch.int32)),
               dict(keep=z(2, 1, 1, dtype=torch.int32)), dict(keep_len=i32(1, 1)),
               dict(dst=i32(0, 0)), dict(to_table=i32(0)), dict(to_table=z(1, 0, dtype=torch.int32)),
               dict(to_table=z(2, 1, dtype=torch.int32)), dict(weights=z(2, 2, 64))],
    }.items():
        f, kw = host_calls()[name]
        for bad in bads:
            with pytest.raises(ops.OpsError):
                f(**{**kw, **bad})
