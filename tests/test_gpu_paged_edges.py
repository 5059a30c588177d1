"""The paged cache operators at their edges."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from paged_model import Cache  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from voxcpm2_b200 import runtime
    return runtime


def unchanged(before, c):
    return all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(before, c.state()))


# ------------------------------------------------------------------ calls that fail as a whole
@pytest.mark.parametrize("length", [-1, 3 * 16 + 1])
def test_compact_with_a_bad_length_changes_nothing(rt, length):
    c = Cache(rt, n_pages=9, n_seqs=3, max_pages=3)
    c.extend([20, 40, 17])
    c.free([1, 0, 0])
    good = c.lens.clone()
    c.lens[2] = length
    before = c.state()
    used = c.compact()
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ] and used.tolist() == [-5]
    assert unchanged(before, c)
    c.status.zero_()
    c.lens.copy_(good)
    assert c.compact().tolist() == [5] and c.status.tolist() == [0]
    assert sorted(c.table[c.table >= 0].tolist()) == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("column,bad", [(0, -1), (1, 40), (2, 2 ** 31 - 1), (2, -2 ** 31), (2, 40)])
def test_fork_of_a_bad_table_changes_nothing(rt, share, column, bad):
    """Parents with a page outside the pool, a full one or the last: no child is made, theirs or another's."""
    c = Cache(rt, n_pages=40, n_seqs=6, max_pages=5)
    c.extend([40, 33, 0, 0, 0, 0])
    good = c.table.clone()
    c.table[0, column] = bad
    before = c.state()
    c.fork([-1, -1, 1, 0, 0, -1], share)
    assert c.status.tolist() == [rt.PAGES_BAD_ID]
    assert unchanged(before, c)
    c.status.zero_()
    c.fork([-1, -1, 1, -1, -1, 1], share)  # nothing of the other parent is looked at
    assert c.status.tolist() == [0] and c.lens.tolist() == [40, 33, 33, 0, 0, 33]
    c.table[0] = good[0]
    c.fork([-1, -1, -1, 0, 0, -1], share)
    assert c.status.tolist() == [0] and c.lens.tolist() == [40, 33, 33, 40, 40, 33]


def test_fork_does_not_look_past_a_parents_end(rt):
    c = Cache(rt, n_pages=20, n_seqs=4, max_pages=5)
    c.extend([32, 0, 0, 0])
    c.table[0, 2:] = 99
    c.fork([-1, 0, 1 << 20, -1])
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ] and c.lens.tolist() == [32, 0, 0, 0]
    c.status.zero_()
    c.fork([-1, 0, -1, 0])
    assert c.status.tolist() == [0] and c.lens.tolist() == [32, 32, 0, 32]


def test_free_leaves_a_sequence_of_bad_length(rt):
    c = Cache(rt, n_pages=20, n_seqs=4, max_pages=3)
    c.extend([20, 33, 40, 5])
    rows, refs = c.table.clone(), c.refs.clone()
    c.lens[1], c.lens[2] = 49, -3
    c.free([1, 1, 1, 0])
    assert c.status.tolist() == [rt.PAGES_BAD_SEQ] and c.lens.tolist() == [0, 49, -3, 5]
    assert c.table[0].tolist() == [-1] * 3 and torch.equal(c.table[1:], rows[1:])
    gone = rows[0, :2].long()
    assert c.refs[gone].tolist() == [0, 0] and int(c.refs.sum()) == int(refs.sum()) - 2
