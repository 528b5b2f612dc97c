"""CPU replay of the norm kernels' rings of rows (``csrc/norm.cu``): a CTA leaves
no bulk copy into its shared memory behind, also where a wait for one has run out."""

import pytest


def ring(rows, depth, late, stops=True, drains=True):
    """Thread 0 of a CTA of so many rows; ``late``: the row whose copy outlasts the wait's limit.
    Rows whose copies are on their way at the end, and rows waited for that were never fetched."""
    issued, seen = set(range(min(depth, rows))), 0
    for n in range(rows):
        if seen == n:
            seen += n != late
        if (seen > n or not stops) and n + depth < rows:
            issued.add(n + depth)
    drained = set(range(seen, min(rows, seen + depth))) if drains else set()
    return issued - set(range(seen)) - drained, drained - issued


CASES = [(rows, depth, late) for depth in (1, 2, 3) for rows in (1, 2, 3, 4, 9) for late in (None, *range(rows))]


@pytest.mark.parametrize("rows, depth, late", CASES)
def test_no_copy_outlives_the_cta(rows, depth, late):
    flying, idle = ring(rows, depth, late)
    assert not flying and not idle


def test_what_a_ring_without_them_leaves():
    """Without the end of the fetches and the drain, copies are on their way when a CTA goes."""
    assert ring(9, 3, None, stops=False, drains=False) == (set(), set())
    assert ring(9, 3, 4, stops=False, drains=False)[0] == {4, 5, 6, 7, 8}
    assert ring(9, 3, 4, drains=False)[0] == {4, 5, 6}
    assert ring(9, 3, 4, stops=False)[0] == {7, 8}
