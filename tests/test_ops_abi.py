"""Refusals of the permutation and MXFP4 entry points: every bad argument is
answered with a status before anything reaches a GPU."""

from __future__ import annotations

import ctypes

P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1001)
BIG = 1 << 40


def test_sorted_rows_and_sizes(moe):
    lib = moe.load_library()
    assert lib.mrml_moe_sorted_rows(128, 8, 0, 1) == 0
    assert lib.mrml_moe_sorted_rows(128, 8, 64, 1) == 512
    assert lib.mrml_moe_sorted_rows(128, 8, 1, 128) == 8 + 8 * 127
    assert lib.mrml_moe_sorted_rows(16, 2, 100, 16) == 200 + 16 * 15
    for bad in ((0, 8, 1, 1), (8, 0, 1, 1), (8, 2, -1, 1), (8, 2, 1, 0), (8, 2, 1, 129), (8, 64, 1 << 25, 1)):
        assert lib.mrml_moe_sorted_rows(*bad) == -1
    assert lib.mrml_moe_sort_workspace_bytes(128, 8, 64) >= 256
    assert lib.mrml_moe_sort_workspace_bytes(257, 8, 64) == 0
    # 128 rows x 64 columns of a tile: 2 blocks of codes and one group of scales
    assert lib.mrml_moe_mx4_bytes(128, 64, 1) == 2 * 2048 + 512
    assert lib.mrml_moe_mx4_bytes(1, 1, 1) == 2 * 2048 + 512
    assert lib.mrml_moe_mx4_bytes(129, 256, 3) == 3 * 2 * (8 * 2048 + 1024)
    assert lib.mrml_moe_mx4_bytes(0, 256, 3) == 0
    assert lib.mrml_moe_mx4_bytes(4, 0, 1) == 0 and lib.mrml_moe_mx4_bytes(-1, 4, 1) == 0
    assert lib.mrml_moe_mx4_matmul_workspace_bytes(1, 64, 64) >= 256
    assert lib.mrml_moe_mx4_matmul_workspace_bytes(1, 0, 64) == 0
    assert lib.mrml_moe_mx4_linear_workspace_bytes(1, 64, 0) == 0
    assert lib.mrml_moe_mx4_experts_workspace_bytes(2816, 704, 128, 8, 64) > 0
    assert lib.mrml_moe_mx4_experts_workspace_bytes(2816, 704, 257, 8, 64) == 0
    assert lib.mrml_moe_mx4_experts_workspace_bytes(0, 704, 128, 8, 64) == 0


def test_a_workspace_serves_fewer_tokens(moe):
    lib = moe.load_library()
    for K in (1, 2, 8, 64):
        tokens = sorted({max(0, n // K + d) for n in (1, 32, 384, 512, 1024, 8192, 24576, 393216, 1 << 19, 1 << 22)
                         for d in (-1, 0, 1, 2)})
        for size in (lambda T: lib.mrml_moe_sort_workspace_bytes(256, K, T),
                     lambda T: lib.mrml_moe_mx4_experts_workspace_bytes(32, 32, 16, K, T),
                     lambda T: lib.mrml_moe_mx4_linear_workspace_bytes(T, 64, 96)):
            sizes = [size(T) for T in tokens]
            assert sizes == sorted(sizes)


def test_sizes_past_the_index_types_are_refused(moe):
    lib = moe.load_library()
    top = 2**31 - 1
    assert lib.mrml_moe_permute(0, P, top, P, P, top, 2, 4, None) == -2
    assert lib.mrml_moe_permute(0, P, 64, P, P, 64, 2, top, None) == -2
    assert lib.mrml_moe_unpermute(0, P, P, P, P, top, top, 2, 4, None) == -2
    assert lib.mrml_moe_unpermute_grad(0, P, 64, P, P, P, P, P, P, 64, 2, 4, top, None) == -2


def test_permutation_refusals(moe):
    lib = moe.load_library()
    sort = lib.mrml_moe_sort
    assert sort(P, P, P, P, P, 0, 8, 1, 1, P, BIG, None) == -1
    assert sort(P, P, P, P, P, 257, 8, 1, 1, P, BIG, None) == -2
    assert sort(P, P, P, P, P, 8, 65, 1, 1, P, BIG, None) == -2
    assert sort(P, P, P, P, P, 8, 8, 1, 129, P, BIG, None) == -2
    assert sort(P, P, P, P, P, 8, 8, 1, 0, P, BIG, None) == -1
    assert sort(P, P, P, P, P, 8, 64, 1 << 25, 1, P, BIG, None) == -2
    assert sort(None, P, P, P, P, 8, 8, 1, 1, P, BIG, None) == -1
    assert sort(P, None, P, P, P, 8, 8, 0, 1, P, BIG, None) == -1
    assert sort(P, P, P, P, P, 8, 8, 1, 1, None, BIG, None) == -1
    assert sort(P, P, P, P, P, 8, 8, 1, 1, ODD, BIG, None) == -1
    assert sort(P, P, P, P, P, 8, 8, 1, 1, P, 16, None) == -3
    perm = lib.mrml_moe_permute
    assert perm(2, P, 64, P, P, 64, 2, 4, None) == -2  # element type
    assert perm(0, P, 63, P, P, 64, 2, 4, None) == -1  # row stride below H
    assert perm(0, P, 64, P, P, 64, 65, 4, None) == -2
    assert perm(0, P, 64, P, P, 64, 2, -1, None) == -1
    assert perm(0, None, 64, P, P, 64, 2, 4, None) == -1
    assert perm(0, ODD, 64, P, P, 64, 2, 4, None) == -1
    assert perm(30, P, 64, P, ODD, 64, 2, 4, None) == -1
    assert perm(0, None, 64, None, None, 64, 2, 0, None) == 0
    for fn in (lambda *a: lib.mrml_moe_unpermute(a[0], a[1], a[2], P, *a[3:]), lib.mrml_moe_permute_grad):
        assert fn(7, P, P, P, 64, 64, 2, 4, None) == -2
        assert fn(0, P, P, P, 60, 64, 2, 4, None) == -1
        assert fn(0, None, P, P, 64, 64, 2, 4, None) == -1
        assert fn(0, P, None, P, 64, 64, 2, 4, None) == -1
        assert fn(0, P, P, ODD, 64, 64, 2, 4, None) == -1
        assert fn(0, P, P, P, 64, 64, 2, -4, None) == -1
        assert fn(0, P, P, P, 64, 64, 2, 1 << 26, None) == -2
        assert fn(0, None, None, None, 64, 64, 2, 0, None) == 0
    grad = lib.mrml_moe_unpermute_grad
    assert grad(0, P, 64, P, P, P, P, P, P, 64, 2, 4, 7, None) == -1  # fewer rows than pairs
    assert grad(0, P, 64, None, P, P, P, P, P, 64, 2, 4, 8, None) == -1  # dprobs needs rows
    assert grad(0, P, 64, P, P, None, P, P, P, 64, 2, 4, 8, None) == -1  # drows needs pair
    assert grad(0, P, 60, P, P, P, P, P, P, 64, 2, 4, 8, None) == -1
    assert grad(0, None, 64, P, P, P, P, P, P, 64, 2, 4, 8, None) == -1
    assert grad(0, P, 64, P, P, P, P, None, None, 64, 2, 4, 8, None) == 0


def test_mx4_refusals(moe):
    lib = moe.load_library()
    q = lib.mrml_moe_mx4_quantize
    assert q(3, P, 64, 0, P, 4, 64, 1, 0, None) == -2
    assert q(0, P, 63, 0, P, 4, 64, 1, 0, None) == -1
    assert q(0, P, 64, 0, P, -1, 64, 1, 0, None) == -1
    assert q(0, P, 64, 0, P, 4, 0, 1, 0, None) == -1
    assert q(0, P, 64, -1, P, 4, 64, 2, 0, None) == -1
    assert q(0, P, 64, 0, P, 3, 64, 1, 1, None) == -1  # a gated matrix has an even number of rows
    assert q(0, P, 64, 0, P, 4, 64, 1 << 16, 0, None) == -2
    assert q(0, P, 64, 0, ctypes.c_void_p(0x1008), 4, 64, 1, 0, None) == -1
    assert q(30, ODD, 64, 0, P, 4, 64, 1, 0, None) == -1
    assert q(0, None, 64, 0, P, 4, 64, 1, 0, None) == -1
    assert q(2, P, 48, 0, P, 4, 48, 1, 0, None) == -1  # GGUF rows are whole blocks
    assert q(8, P, 96, 0, P, 4, 64, 1, 0, None) == -1  # ... without gaps
    assert q(8, P, 64, 100, P, 4, 64, 2, 0, None) == -1
    assert q(0, None, 64, 0, None, 0, 64, 1, 0, None) == 0
    both = lib.mrml_moe_mx4_quantize_both
    assert both(2, P, 64, P, P, 4, 64, None) == -2
    assert both(0, P, 60, P, P, 4, 64, None) == -1
    assert both(0, P, 64, P, None, 4, 64, None) == -1
    assert both(0, P, 64, P, ODD, 4, 64, None) == -1
    assert both(0, None, 64, None, None, 0, 64, None) == 0
    dq = lib.mrml_moe_mx4_dequantize
    assert dq(8, P, P, 64, 0, 4, 64, 1, 0, None) == -2
    assert dq(0, P, P, 60, 0, 4, 64, 1, 0, None) == -1
    assert dq(0, P, P, 64, 0, 5, 64, 1, 1, None) == -1
    assert dq(0, ODD, P, 64, 0, 4, 64, 1, 0, None) == -1
    mm = lib.mrml_moe_mx4_matmul
    assert mm(2, P, P, P, 64, 4, 64, 64, P, BIG, None) == -2
    assert mm(0, P, P, P, 60, 4, 64, 64, P, BIG, None) == -1
    assert mm(0, P, P, P, 64, 4, 64, 0, P, BIG, None) == -1
    assert mm(0, P, None, P, 64, 4, 64, 64, P, BIG, None) == -1
    assert mm(0, ODD, P, P, 64, 4, 64, 64, P, BIG, None) == -1
    assert mm(0, P, P, P, 64, 4, 64, 64, P, 8, None) == -3
    assert mm(0, P, P, P, 64, 4, 64, 64, ODD, BIG, None) == -1
    assert mm(0, None, None, None, 64, 0, 64, 64, None, 0, None) == 0
    lin = lib.mrml_moe_mx4_linear
    assert lin(0, P, 60, P, P, 64, 4, 64, 64, P, BIG, None) == -1
    assert lin(0, P, 64, P, P, 60, 4, 64, 64, P, BIG, None) == -1
    assert lin(0, P, 64, ODD, P, 64, 4, 64, 64, P, BIG, None) == -1
    assert lin(0, P, 64, P, P, 64, 4, 64, 64, P, 300, None) == -3
    ex = lib.mrml_moe_mx4_experts
    ok = [30, P, P, P, P, None, P, 64, P, 64, 64, 32, 8, 2, 4, P, BIG, None]

    def refuse(status, **change):
        names = "type gate_up down ids probs scale x ldx out ldo H I E K T ws bytes stream".split()
        a = list(ok)
        for k, v in change.items():
            a[names.index(k)] = v
        assert ex(*a) == status, change

    refuse(-2, type=2)
    refuse(-2, E=257)
    refuse(-2, K=65)
    refuse(-1, H=0)
    refuse(-1, I=0)
    refuse(-1, T=-1)
    refuse(-1, ldx=63)
    refuse(-1, ldo=63)
    refuse(-1, gate_up=ODD)
    refuse(-1, down=None)
    refuse(-1, ids=None)
    refuse(-1, x=ODD)
    refuse(-1, ws=ODD)
    refuse(-3, bytes=256)
    refuse(0, T=0, x=None, out=None, ws=None)
