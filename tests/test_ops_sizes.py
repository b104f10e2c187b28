"""Sizes that the permutation and MXFP4 operators report for shapes that they refuse (no GPU needed)."""

from __future__ import annotations

import pytest

TOP = 2**31 - 1


@pytest.mark.parametrize("shape", [(1 << 24, 65, 1 << 19, 128), (TOP, 64, 1 << 20, 128), (1 << 25, 1, 1 << 26, 64)])
def test_more_sorted_rows_than_an_index_holds_are_refused(moe, shape):
    assert moe.load_library().mrml_moe_sorted_rows(*shape) == -1
    with pytest.raises(moe.MoeError):
        moe.sorted_rows(*shape)


def test_the_largest_sorts_have_a_size(moe):
    lib = moe.load_library()
    assert lib.mrml_moe_sorted_rows(256, 64, 1 << 20, 128) == (1 << 26) + 256 * 127
    assert lib.mrml_moe_sorted_rows(1 << 24, 1, 1 << 24, 127) == (1 << 24) * 127
