"""GPU test of the paged prep's rotary widths: every token of a wave turns by its own
position, however few lanes rotate. Tolerances are test_gpu_paged.py's."""
import pytest

torch = pytest.importorskip("torch")

import paged_oracle as po  # noqa: E402
import test_gpu_paged as gp  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rot", [8, 16, 32, 64])
def test_prep_turns_each_token_by_its_own_position(rot, e4m3):
    o = gp.ops()
    Hq, Hkv, N = 4, 2, 70
    pages = gp.pool(501, 3, Hkv, e4m3)
    g = torch.Generator().manual_seed(502)
    proj = torch.randn(N, Hq * 512 + Hkv * 512, generator=g).bfloat16()
    qw, kw = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    pos = torch.randint(0, 600, (N,), generator=g, dtype=torch.int32)
    rope = o.rope_table(1e7, rot, 600)
    q_out = torch.zeros(N, Hq, D, dtype=torch.bfloat16, device="cuda")
    o.attn_prep_paged(proj.cuda(), qw.cuda(), kw.cuda(), pos.cuda(), gp.i32([0, N]), gp.i32([N]),
                      gp.i32([[2, 0]]), Hq, rot, rope, 1e-6, gp.Q_SCALE, q_out, pages)
    torch.cuda.synchronize()
    cs = rope.cpu().double()[pos.long()][:, None]
    x = proj.double()
    q = po.norm_rope(x[:, :Hq * 512].view(N, Hq, 512)[..., :D], qw.double(), cs[..., 0],
                     cs[..., 1], rot, 1e-6) * gp.Q_SCALE
    k = po.norm_rope(x[:, Hq * 512:Hq * 512 + Hkv * D].view(N, Hkv, D), kw.double(), cs[..., 0],
                     cs[..., 1], rot, 1e-6)
    assert ((q_out.cpu().double() - q).abs() <= q.abs() * 2 ** -8 +
            1e-5 * q.abs().amax(-1, keepdim=True)).all()
    got, _ = gp.values(pages)
    got = torch.cat([got[2], got[0]], 1).transpose(0, 1)[:N]
    if e4m3:
        kq, ks = po.quantise(k, 2)
        assert torch.equal(got, kq * ks[..., None])
    else:
        assert ((got - k).abs() <= k.abs() * 2 ** -8 +
                1e-5 * k.abs().amax(-1, keepdim=True)).all()
