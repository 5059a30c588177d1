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
