"""Drafts of a text generator: continuations found in the history, merged into a tree."""
from noise_b200.generate import grow, repeated


def test_repeated():
    assert repeated([1, 2, 3, 4, 1, 2], 2) == [[3, 4]]
    assert repeated([1, 2, 3, 1, 2, 4, 1, 2], 3) == [[4, 1, 2], [3, 1, 2]]
    assert repeated([1, 2, 3, 1, 2, 4, 1, 2], 3, branches=1) == [[4, 1, 2]]
    assert repeated([1, 1, 1], 2) == [[1]]
    assert repeated([1], 2) == [] and repeated([1, 2], 2) == [] and repeated([1, 2, 3], 2) == []


def test_grow():
    assert grow(9, [], 1) == ([9], [-1])
    assert grow(9, [[1]], 1) == ([9], [-1])
    assert grow(9, [], 3) == ([9, 0, 0], [-1, -2, -2])
    assert grow(9, [[4, 1, 2], [3, 1], [4, 1, 5]], 8) == ([9, 4, 1, 2, 3, 1, 5, 0], [-1, 0, 1, 2, 0, 4, 2, -2])
    assert grow(9, [[4, 1, 2], [4, 7]], 4) == ([9, 4, 1, 2], [-1, 0, 1, 2])
