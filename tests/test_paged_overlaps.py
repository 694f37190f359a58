"""Arrays of a call that may not overlap, refused on the CPU by the host's checks before
anything is launched. The base cases are test_paged_more_args.py's."""
import pytest

pytest.importorskip("torch")

from test_paged_args import FAKE, INVALID  # noqa: E402
from test_paged_more_args import KEEP, SELECT, WEIGHTS, call  # noqa: E402


@pytest.mark.parametrize("at", [0, 4, 28, -4, -20])
def test_keep_refuses_a_goal_that_is_its_source(at):
    """4 sequences of 2 pages to 3 each: in place is to_table NULL."""
    bad = dict(B=4, to_table=FAKE + at, to_pages=3)
    st, msg = call(KEEP, **bad)
    assert st == INVALID and "to_table" in msg


@pytest.mark.parametrize("at", [0, 32, -48])
def test_keep_takes_tables_that_do_not_overlap(at):
    """Nothing to keep: no launch. No sequence: no array."""
    assert call(KEEP, B=4 if at else 0, to_table=FAKE + at, to_pages=3, max_keep=0)[0] == 0


@pytest.mark.parametrize("at", [4, -4, 28, -28])
def test_select_refuses_lengths_that_it_writes_over(at):
    """A kv-head writes what the others of its sequence, or of the next, still read."""
    st, msg = call(SELECT, B=8, kv_len=FAKE, keep_len=FAKE + at)
    assert st == INVALID and "keep_len" in msg


@pytest.mark.parametrize("at", [4, -4, 256 * 8 - 4, 4 - 256 * 8])
def test_weights_refuse_what_was_written_over_before_it_is_read(at):
    """4 pages of 2 kv-heads: weights of one slot where prev has another's."""
    st, msg = call(WEIGHTS, N=1, B=1, prev=FAKE + at)
    assert st == INVALID and "prev" in msg


def test_weights_take_prev_beside_them():
    """No rows: no launch."""
    for at in (0, 256 * 8, -256 * 8):
        assert call(WEIGHTS, B=1, prev=FAKE + at)[0] == 0
