"""pages.compact where others than the table's rows hold pages: as a row of the call they learn where those went."""
import pytest
import torch

import pages_reference as R

pytestmark = pytest.mark.gpu


def test_kept_pages_are_named_by_a_row_of_the_call(dev):
    from uwc_amd import pages as P
    cs = [R.cache(40, 2, 32, 16, torch.Generator().manual_seed(i), dev) for i in range(2)]
    table, kept = [[30, 7, 21, -1], [30, 12, -1, -1]], [39, 30, 25]  # one page belongs to a row and is kept too
    refs = [0] * 40
    for p in [p for r in table for p in r if p >= 0] + kept:
        refs[p] += 1
    before = [tuple(x.clone() for x in c) for c in cs]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t, n = P.compact(cs, ints(table + [kept + [-1]]), ints(refs))
    was, now = table + [kept + [-1]], t.tolist()
    assert sorted({p for r in now for p in r if p >= 0}) == list(range(6)) and n[6:].sum() == 0
    for a, b in zip(sum(was, []), sum(now, [])):
        assert (a < 0) == (b < 0)
        if a >= 0:
            assert n[b] == refs[a] and all(torch.equal(x[b], y[a]) for c, o in zip(cs, before) for x, y in zip(c, o))
