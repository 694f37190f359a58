"""GPU tests of attention weights by key: up to 128 rows, waves of several pages, weights
at the ends of fp32; against the float64 form of evict_oracle.py."""
import pytest

torch = pytest.importorskip("torch")

import paged_oracle as po  # noqa: E402
import test_gpu_evict as ge  # noqa: E402
import test_gpu_paged as gp  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", [
    # 33 to 64 rows, 65, 68, 100, 128
    (16, 4, [(9, 300), (16, 70), (1, 64)]), (5, 1, [(13, 700), (2, 64)]), (16, 4, [(17, 300)]),
    (4, 4, [(100, 700), (65, 66), (0, 9), (1, 130)]), (16, 4, [(32, 1000), (20, 70), (1, 5)]),
    (8, 2, [(32, 20), (25, 128)])])
def test_weights_of_some_rows(Hq, Hkv, lens, e4m3):
    c = ge.fill(gp.attention_case(661, Hq, Hkv, e4m3, lens), 662)
    ge.check_weights(c, ge.weigh(c))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hkv,lens,B", [
    # waves of two pages; of 66, more than they have ids of at a time
    (4, [(2, 1400), (8, 70), (1, 1100)], 12500), (4, [(1, 264 * PAGE - 5), (3, 9000)], 66000)])
def test_weights_of_many_sequences_without_rows(Hkv, lens, B, e4m3):
    """For so many that a wave takes several pages; those without rows are left out."""
    o = gp.ops()
    c = ge.fill(gp.attention_case(671, Hkv, Hkv, e4m3, lens), 672)
    tiles = -(-c["max_kv"] // PAGE)
    assert B * Hkv * tiles > 1 << 20
    tab = torch.full((B, tiles), -1, dtype=torch.int32, device="cuda")
    tab[:len(lens)] = gp.i32(c["tab"])
    qs = torch.full((B + 1,), c["qs"][-1], dtype=torch.int32, device="cuda")
    qs[:len(lens) + 1] = gp.i32(c["qs"])
    kv = torch.full((B,), 64, dtype=torch.int32, device="cuda")
    kv[:len(lens)] = gp.i32(c["kv_len"])
    w = c["w"].cuda()
    o.kv_weights(c["q"].cuda(), c["lse"].cuda(), c["pages"], tab, qs, kv, c["max_q"], c["max_kv"],
                 w, prev=c["prev"].cuda())
    torch.cuda.synchronize()
    ge.check_weights(c, w.cpu())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lens", [[(200, 600)], [(16, 600)]])
@pytest.mark.parametrize("most,lse", [(-26.0, None), (128.0, 31.0), (3.0, -31.0)])
def test_weights_at_the_ends_of_fp32(lens, most, lse, e4m3):
    """Weights of 2^-110, and of 2^97 by another lse than the rows' own: q.k alone is past
    the ends of fp32's exponent."""
    c = gp.attention_case(681, 8, 2, e4m3, lens)
    k = torch.zeros(c["pages"].k.shape)
    k[..., 0] = most
    k[:, :, 5::16, 0] = -128.0
    c["pages"].k.copy_(k.to(c["pages"].k.dtype))
    if e4m3:
        c["pages"].k_scale.fill_(1.0)
    c["q"].zero_()
    c["q"][..., 0] = 1.0
    c = ge.fill(c, 682)
    if lse is not None:
        c["lse"].fill_(lse)
    for name in ("prev", "w"):
        c[name].zero_()
    ge.check_weights(c, ge.weigh(c))
