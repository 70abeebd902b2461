"""tree_shape on the CPU: level-by-level numbering, refusals."""

import pytest

from myinfer_b200.generate import tree_shape


def test_levels():
    assert tree_shape((1, 1)) == [[-1], [0], [1]]
    assert tree_shape((3, 2)) == [[-1], [0, 0, 0], [1, 1, 2, 2, 3, 3]]
    flat = [p for lv in tree_shape((4, 2, 1, 1)) for p in lv]
    assert len(flat) == 1 + 4 + 8 + 8 + 8 and all(p < i for i, p in enumerate(flat))


@pytest.mark.parametrize("widths", [(), (0,), (2, -1), (64,), (8, 8)])
def test_refusals(widths):
    with pytest.raises(ValueError):
        tree_shape(widths)
