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


# H, I, E, K, T
REFUSED = [(TOP, 64, 8, 2, 4), ((1 << 24) + 1, 64, 8, 2, 4), (64, TOP, 8, 2, 4), (64, 1 << 30, 8, 2, 4), (64, (1 << 24) + 1, 8, 2, 4),
           (64, 64, 8, 65, 4), (64, 64, 257, 2, 4), (64, 64, 8, 2, -1), (64, 0, 8, 2, 4), (1 << 24, 1 << 24, 8, 64, 1 << 20)]


@pytest.mark.parametrize("shape", REFUSED)
def test_a_layer_that_is_refused_has_no_workspace_size(moe, shape):
    lib = moe.load_library()
    H, I, E, K, T = shape
    p = 0x1000
    assert lib.mrml_moe_mx4_experts_workspace_bytes(*shape) == 0
    assert lib.mrml_moe_mx4_experts(30, p, p, p, p, None, p, H, p, H, H, I, E, K, T, p, 1 << 62, None) in (-1, -2)


def test_the_largest_layers_have_a_size(moe):
    lib = moe.load_library()
    # 16 rows of down products in 32 bits (a tile of 128 per expert that has one), and the quantised rows beside them
    for H, I in ((1 << 24, 32), (32, 1 << 24)):
        n = 16 + 8 * 127
        assert lib.mrml_moe_mx4_experts_workspace_bytes(H, I, 8, 2, 8) > n * H * 4 + 8 * 128 * (H + I) // 2
