"""GPU tests of draft trees of a middling number of rows whose workgroups have long pieces
of the key tiles (test_paged_tree_cases.py checks on the CPU that they are), and of those
with up to 32 rows, against the float64 forms of evict_oracle.py."""
import random

import pytest

torch = pytest.importorskip("torch")

import paged_oracle as po  # noqa: E402
import test_gpu_paged as gp  # noqa: E402
import test_gpu_paged_tree as gt  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = po.PAGE, po.D

# Many kv-heads leave a kv-head few workgroups, so that a piece is long.
LONG = [
    # (Hq, Hkv, [(drafted tokens, keys)])
    (64, 64, [(40, 2000), (20, 130), (0, 300), (64, 1500)]),
    (64, 64, [(20, 2000), (17, 130), (32, 1501)]),             # up to 32 rows
    (192, 64, [(16, 1990), (9, 130), (21, 1100), (1, 64)]),    # three heads a group
    (256, 256, [(20, 4300), (3, 2), (5, 0), (17, 200)]),       # a piece of more than 64 tiles
    (256, 256, [(64, 4300), (33, 200)]),
]
# (page by page, how much higher the scores are)
LEVELS = [0., 2., 5., 9., 13., 18., 20., 40., 44., 60., 72., 88.]
RISING = [(64, 64, [(40, 1900), (33, 1100)]), (64, 64, [(20, 1900), (32, 1100)])]
# up to 32 rows
SMALL = [(16, 4, [(5, 300), (8, 70)]), (8, 1, [(3, 700)]), (4, 1, [(8, 8), (5, 3), (0, 40), (6, 0)]),
         (6, 2, [(7, 300)] * 70), (16, 1, [(2, 130), (1, 64)])]


def repeated(seed, Hq, Hkv, e4m3, lens, pages=9):
    """A case over a pool of few pages, each of which the sequences have many times."""
    c = gt.tree_case(seed, Hq, Hkv, e4m3, [(n, min(kv, 64)) for n, kv in lens])
    r = random.Random(seed)
    c["pages"] = gp.pool(seed, pages, Hkv, e4m3)
    need = [-(-kv // PAGE) for _, kv in lens]
    c["tab"] = [[r.randrange(pages) for _ in range(n)] + [-1] * (max(need) - n) for n in need]
    c["kv_len"] = [kv for _, kv in lens]
    c["max_kv"] = max(c["kv_len"])
    return c


def check(c, got, lse):
    """gt.check, whose oracle takes a key at least: one that no row sees where there is none."""
    empty = [kv == 0 for kv in c["kv_len"]]
    seen = gt.tree_seen(c)
    few = {**c, "kv_len": [kv or 1 for kv in c["kv_len"]],
           "tab": [[0] + row[1:] if no else row for row, no in zip(c["tab"], empty)]}
    gt.check(few, got, lse, lambda b, p0, ql, kv: torch.zeros(ql, kv, dtype=torch.bool)
             if empty[b] else seen(b, p0, ql, kv))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", LONG)
def test_long_pieces_match_oracle(Hq, Hkv, lens, e4m3):
    c = repeated(501, Hq, Hkv, e4m3, lens)
    c["tab"][0][5], c["tab"][0][17] = -1, c["pages"].num_pages  # two that are not there
    got, lse = gt.run(c, c["tree"])
    check(c, got, lse)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("order", ["up", "down", "turns", "any"])
@pytest.mark.parametrize("Hq,Hkv,lens", RISING)
def test_scores_move_the_reference_within_a_piece(Hq, Hkv, lens, order, e4m3):
    """From tile to tile, by less and by more than lets it stay, for some rows and not for
    others."""
    c = repeated(511, Hq, Hkv, e4m3, lens, pages=len(LEVELS))
    k = torch.zeros(c["pages"].k.shape)
    k[..., 0] = torch.tensor(LEVELS)[:, None, None]
    k[..., 1] = torch.arange(PAGE) / 64
    c["pages"].k.copy_(k.to(c["pages"].k.dtype))
    if e4m3:
        c["pages"].k_scale.fill_(1.0)
    r, n = random.Random(512), len(LEVELS)
    for row, (_, kv) in zip(c["tab"], lens):
        for i in range(-(-kv // PAGE)):
            at = i * n // -(-kv // PAGE)
            row[i] = {"up": at, "down": n - 1 - at, "turns": (5 * i) % n, "any": r.randrange(n)}[order]
    g = torch.Generator().manual_seed(513)
    c["q"][..., 0] = torch.tensor([1.0, 0.5, 0.25, -0.5, -1.0])[
        torch.randint(0, 5, (c["N"], Hq), generator=g)].bfloat16()
    c["q"][..., 1] = 1.0
    got, lse = gt.run(c, c["tree"])
    check(c, got, lse)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("Hq,Hkv,lens", SMALL)
def test_up_to_32_rows_match_oracle(Hq, Hkv, lens, e4m3):
    c = gt.tree_case(521, Hq, Hkv, e4m3, lens)
    got, lse = gt.run(c, c["tree"])
    check(c, got, lse)


@pytest.mark.parametrize("e4m3", [False, True])
def test_up_to_32_rows_as_others_are_tested(e4m3):
    """Hidden keys, rows that see nothing, missing pages, large scores."""
    gt.test_trees_ignore_what_no_row_sees([(5, 300), (8, 70), (7, 64)], e4m3)
    gt.test_rows_that_see_nothing_give_zero([(7, 7), (8, 100)], e4m3)
    gt.test_trees_skip_pages_that_are_not_there([(8, 400), (5, 70)], e4m3)
    gt.test_trees_past_max_q([(20, 300), (2, 90), (6, 64)], 8, e4m3)
    for scale in (900.0, -900.0):
        gt.test_trees_of_large_scores([(8, 300), (6, 70)], scale, e4m3)
