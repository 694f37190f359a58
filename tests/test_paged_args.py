"""Refusals of the paged K/V cache's entry points, on the CPU: every call here
is turned away by the host's checks before anything is launched."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from cujev import ops  # noqa: E402

FAKE = 1 << 20  # a well-aligned address that nothing may touch
INVALID, CAPACITY = 1, 6


def call(name, **changes):
    args = dict(BASE[name])
    assert set(changes) <= set(args), changes
    args.update(changes)
    lib = ops.load()
    st = getattr(lib, name)(*args.values())
    return st, lib.cujev_ops_last_error().decode()


POOL = dict(kv_type=1, k_pages=FAKE, vt_pages=FAKE, k_scale=FAKE, v_scale=FAKE, num_pages=4)
BASE = {
    "cujev_op_attn_prep_paged": dict(
        proj=FAKE, proj_stride=5120, q_norm_w=FAKE, k_norm_w=FAKE, pos=FAKE, q_start=FAKE,
        kv_len=FAKE, page_table=FAKE, max_pages=2, B=0, N=0, Hq=8, Hkv=2, rot=64, rope_table=FAKE,
        npos=128, eps=1e-6, q_scale=0.09, q_out=FAKE, **POOL, stream=None),
    "cujev_op_kv_page_read": dict(
        **POOL, page_table=FAKE, max_pages=2, kv_len=FAKE, B=0, max_kv=128, Hkv=2, k_cache=FAKE,
        vt_cache=FAKE, cache_stride=192, stream=None),
    "cujev_op_attention_paged": dict(
        q=FAKE, gate=FAKE, gate_tok_stride=5120, gate_head_stride=512, **POOL, q_start=FAKE,
        kv_len=FAKE, page_table=FAKE, max_pages=2, B=0, N=0, max_q=1, max_kv=128, Hq=8, Hkv=2,
        window=0, sinks=0, out=FAKE, ws=None, ws_bytes=0, stream=None),
}
READ, PREP, ATTN = "cujev_op_kv_page_read", "cujev_op_attn_prep_paged", "cujev_op_attention_paged"


def test_argument_order_is_the_headers():
    for name, args in BASE.items():
        assert len(args) == len(ops._SIGS[name])


@pytest.mark.parametrize("name", [PREP, READ, ATTN])
def test_an_empty_call_does_nothing(name):
    assert call(name)[0] == 0


BAD_POOL = [dict(kv_type=2), dict(kv_type=-1), dict(k_pages=None), dict(vt_pages=None),
            dict(k_pages=FAKE + 8), dict(vt_pages=FAKE + 2), dict(k_scale=None),
            dict(v_scale=None), dict(v_scale=FAKE + 4), dict(num_pages=0), dict(num_pages=-1),
            dict(Hkv=0), dict(max_pages=0), dict(max_pages=(1 << 22) + 1), dict(B=-1),
            dict(B=1, page_table=None), dict(B=1, kv_len=None)]


@pytest.mark.parametrize("name", [PREP, READ, ATTN])
@pytest.mark.parametrize("bad", BAD_POOL, ids=str)
def test_pool_and_table_are_checked(name, bad):
    st, msg = call(name, **bad)
    assert st == INVALID and name[9:] in msg


@pytest.mark.parametrize("bad", [
    dict(N=-1), dict(Hq=7), dict(Hq=0), dict(Hq=34), dict(Hq=1 << 30, Hkv=1 << 29), dict(rot=0), dict(rot=24), dict(rot=128),
    dict(npos=0), dict(proj_stride=5119), dict(proj_stride=5121), dict(proj=FAKE + 4),
    dict(q_out=FAKE + 4), dict(q_norm_w=FAKE + 4), dict(rope_table=FAKE + 8),
    dict(N=1, B=1, proj=None), dict(N=1, B=1, q_start=None), dict(N=1, B=1, q_out=None),
    dict(N=1, B=1, pos=None), dict(N=1, B=1, rope_table=None), dict(N=1, B=1, q_norm_w=None),
    dict(N=1, B=1, k_norm_w=None)], ids=str)
def test_prep_refuses(bad):
    assert call(PREP, **bad)[0] == INVALID


@pytest.mark.parametrize("bad", [
    dict(max_kv=-1), dict(max_kv=129), dict(cache_stride=128), dict(cache_stride=200),
    dict(B=1, k_cache=None), dict(B=1, vt_cache=FAKE + 8), dict(B=70000)], ids=str)
def test_read_refuses(bad):
    assert call(READ, **bad)[0] == INVALID


@pytest.mark.parametrize("bad", [
    dict(N=-1), dict(max_q=-1), dict(max_kv=-1), dict(max_kv=129), dict(Hq=7), dict(Hq=34),
    dict(Hq=8200, Hkv=4100),
    dict(window=-1), dict(window=8, sinks=-1), dict(sinks=4), dict(q=FAKE + 8), dict(out=FAKE + 8),
    dict(gate=FAKE + 2), dict(gate_tok_stride=5121), dict(gate_head_stride=2),
    dict(N=1, B=1, q=None), dict(N=1, B=1, q_start=None), dict(N=1, B=1, out=None)], ids=str)
def test_attention_refuses(bad):
    assert call(ATTN, **bad)[0] == INVALID


def test_bindings_refuse_wrong_tensors():
    k = torch.zeros(2, 1, 64, 256, dtype=torch.bfloat16)
    vt = torch.zeros(2, 1, 256, 64, dtype=torch.bfloat16)
    sc = torch.zeros(2, 1, 64)
    f8 = torch.float8_e4m3fn
    pages = ops.KvPages(k, vt)
    ops.KvPages(k.to(f8), vt.to(f8), sc, sc)
    for args in [(k, vt, sc, sc), (k.half(), vt.half()), (k, vt[:1]), (k, vt.transpose(2, 3)),
                 (k.to(f8), vt.to(f8)), (k.to(f8), vt, sc, sc), (k[..., :128], vt),
                 (k.to(f8), vt.to(f8), sc.double(), sc)]:
        with pytest.raises(ops.OpsError):
            ops.KvPages(*args)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    q, out = torch.zeros(1, 4, 256).bfloat16(), torch.zeros(1, 1024).bfloat16()
    good = dict(q=q, gate=None, gate_tok_stride=0, gate_head_stride=0, pages=pages,
                page_table=i32(0)[None], q_start=i32(0, 1), kv_len=i32(1), max_q=1, max_kv=1,
                out=out)
    for bad in [dict(q=q.float()), dict(q=q[..., :128]), dict(out=out[:, :512]),
                dict(kv_len=i32(1, 2)), dict(q_start=i32(0)), dict(page_table=i32(0)),
                dict(kv_len=torch.tensor([1])), dict(ws=torch.zeros(4)),
                dict(gate=q.float()), dict(gate=q, gate_tok_stride=1024, gate_head_stride=512),
                dict(gate=q, gate_tok_stride=-4), dict(q=q[0]), dict(max_kv=2 ** 32 + 1),
                dict(max_q=-1), dict(window=2 ** 31)]:
        with pytest.raises(ops.OpsError):
            ops.attention_paged(**{**good, **bad})
    kc, vc = torch.zeros(1, 1, 128, 256).bfloat16(), torch.zeros(1, 1, 256, 128).bfloat16()
    for a, b in [(kc[0], vc), (kc.flatten(), vc), (kc, vc[..., :64]), (kc.float(), vc)]:
        with pytest.raises(ops.OpsError):
            ops.kv_page_read(pages, i32(0)[None], i32(1), 1, a, b)
    for max_kv in (2 ** 32 + 1, -1):
        with pytest.raises(ops.OpsError):
            ops.kv_page_read(pages, i32(0)[None], i32(1), max_kv, kc, vc)
        with pytest.raises(ops.OpsError):
            ops.attention_paged_ws_bytes(1, 1, 1, max_kv, 4, 1)
    w = torch.ones(256)
    prep = dict(proj=torch.zeros(1, 4 * 512 + 512).bfloat16(), q_norm_w=w, k_norm_w=w, pos=i32(0),
                q_start=i32(0, 1), kv_len=i32(1), page_table=i32(0)[None], Hq=4, rot=64,
                rope=torch.zeros(8, 32, 2), eps=1e-6, q_scale=0.1, q_out=q, pages=pages)
    for bad in [dict(proj=prep["proj"].float()), dict(proj=prep["proj"][:, :2048]),
                dict(proj=prep["proj"][0]),
                dict(pos=i32(0, 1)), dict(rope=torch.zeros(8, 16, 2)), dict(q_out=q[:, :2]),
                dict(q_norm_w=w.bfloat16()), dict(k_norm_w=w[:128])]:
        with pytest.raises(ops.OpsError):
            ops.attn_prep_paged(**{**prep, **bad})


def host_calls(e4m3):
    """Calls of the three operators that are right but for the memory: all on the CPU."""
    t = torch.float8_e4m3fn if e4m3 else torch.bfloat16
    sc = [torch.ones(2, 1, 64) for _ in range(2 * e4m3)]
    pages = ops.KvPages(torch.zeros(2, 1, 64, 256).to(t), torch.zeros(2, 1, 256, 64).to(t), *sc)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    q, w, seqs = bf(1, 4, 256), torch.ones(256), dict(kv_len=i32(1), page_table=i32(0)[None])
    return {
        PREP: lambda: ops.attn_prep_paged(
            proj=bf(1, 2560), q_norm_w=w, k_norm_w=w, pos=i32(0), q_start=i32(0, 1), Hq=4, rot=64,
            rope=torch.zeros(8, 32, 2), eps=1e-6, q_scale=0.1, q_out=q, pages=pages, **seqs),
        READ: lambda: ops.kv_page_read(pages, max_kv=1, k_cache=bf(1, 1, 128, 256),
                                       vt_cache=bf(1, 1, 256, 128), **seqs),
        ATTN: lambda: ops.attention_paged(
            q=q, gate=None, gate_tok_stride=0, gate_head_stride=0, pages=pages,
            q_start=i32(0, 1), max_q=1, max_kv=1, out=bf(1, 1024), **seqs)}


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("name", [PREP, READ, ATTN])
def test_bindings_refuse_tensors_in_host_memory(name, e4m3, monkeypatch):
    """Device index -1 is the CPU's, and torch reads it as the current GPU's: such a
    call would launch with host pointers. Nothing here can: the library is a stand-in."""
    reached = []

    class Library:
        def __getattr__(self, symbol):
            return lambda *args: reached.append(symbol) or 0

    monkeypatch.setattr(ops, "_lib", Library())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0, raising=False)
    with pytest.raises(ops.OpsError, match="host memory"):
        host_calls(e4m3)[name]()
    assert not reached


def test_a_workspace_of_the_largest_call_serves_the_smaller_ones():
    """A prompt of 4096 merges nothing, the chunks and single tokens after it do."""
    size = lambda N, B, max_q, max_kv, **kw: ops.attention_paged_ws_bytes(N, B, max_q, max_kv, 16,
                                                                         4, **kw)
    most = size(4096, 64, 4096, 8192)
    assert 0 < most < 35 << 20
    for N, B, max_q in [(4096, 1, 4096), (512, 1, 512), (64, 64, 1), (1, 1, 1), (2047, 64, 1024),
                        (2048, 64, 1024)]:
        for kw in (dict(), dict(window=512, sinks=4), dict(e4m3=True)):
            for max_kv in (100, 1000, 8192):
                assert size(N, B, max_q, max_kv, **kw) <= most


def test_prep_refuses_strides_that_an_int_does_not_hold():
    """ctypes cuts them: rows 2^32 + 2560 values apart would be read as 2560 apart. (The
    memory is asked for and never touched.)"""
    pages = ops.KvPages(torch.zeros(2, 1, 64, 256).bfloat16(), torch.zeros(2, 1, 256, 64).bfloat16())
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    far = 2 ** 32 + 2560
    proj = torch.empty(far + 2560, dtype=torch.bfloat16).as_strided((2, 2560), (far, 1))
    w = torch.ones(256)
    with pytest.raises(ops.OpsError, match="stride of proj"):
        ops.attn_prep_paged(proj, w, w, i32(0, 1), i32(0, 2), i32(2), i32(0)[None], 4, 64,
                            torch.zeros(8, 32, 2), 1e-6, 0.1,
                            torch.zeros(2, 4, 256).bfloat16(), pages)


def test_a_pool_keeps_the_tensors_that_were_checked():
    """The calls go by the addresses taken then: another tensor in a tensor's place would
    be passed over, and the memory of the old one written to after it was freed."""
    f8, sc = torch.float8_e4m3fn, torch.ones(2, 1, 64)
    k, vt = torch.zeros(2, 1, 64, 256).to(f8), torch.zeros(2, 1, 256, 64).to(f8)
    pages = ops.KvPages(k, vt, sc, sc.clone())
    for name in ("k", "vt", "k_scale", "v_scale"):
        with pytest.raises(AttributeError):
            setattr(pages, name, getattr(pages, name).clone())
    assert pages.k is k and pages.vt is vt and pages.k_scale is sc
    assert pages.args == (1, k.data_ptr(), vt.data_ptr(), sc.data_ptr(),
                          pages.v_scale.data_ptr(), 2)


@pytest.mark.parametrize("big", [dict(N=1 << 26, B=1), dict(N=1 << 28, B=1 << 28),
                                 dict(N=1 << 26, B=1, kv_type=0)], ids=str)
def test_prep_refuses_more_work_items_than_a_launch_may_have(big):
    """2^32 and more, in a grid that is still an int."""
    st, msg = call(PREP, **big)
    assert st == INVALID and "unsupported shape" in msg


@pytest.mark.parametrize("big", [
    dict(N=1 << 23, B=1 << 21, max_q=4),  # 4 workgroups of 256 for each of 2^22 units
    dict(N=1 << 23, B=(1 << 21) + 1, max_q=1)], ids=str)
def test_attention_refuses_more_work_items_than_a_launch_may_have(big):
    """Before the attention itself has run, not after it."""
    st, msg = call(ATTN, **{**big, "ws": FAKE, "ws_bytes": 1 << 40})
    assert st == INVALID and "unsupported shape" in msg
