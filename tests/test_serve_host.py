"""The page pool's bookkeeping (uwc_b200.serve.PagePool), without a device."""
import pytest


def test_pages_are_taken_kept_and_given_back():
    from uwc_b200._lib import UWCError
    from uwc_b200.serve import PagePool
    p = PagePool(pages=5, slots=3, width=3, page_size=16)
    assert p.table().tolist() == [[-1] * 3] * 3
    assert p.missing(0, 0) == 0 and not p.hold(0, 0)
    assert p.hold(0, 1) and not p.hold(0, 16) and p.hold(0, 17)        # a page at each 16 tokens
    assert p.hold(2, 48)
    held = p.rows[0] + p.rows[2]
    assert len(set(held)) == 5 and not p.free
    with pytest.raises(UWCError):
        p.hold(1, 1)
    with pytest.raises(ValueError):
        p.hold(2, 49)                                                 # wider than the table
    assert p.table().tolist() == [p.rows[0] + [-1], [-1] * 3, p.rows[2]]
    p.give_back(2)
    assert p.hold(1, 48) and set(p.rows[1]).isdisjoint(p.rows[0])
    assert p.table()[2].tolist() == [-1] * 3
