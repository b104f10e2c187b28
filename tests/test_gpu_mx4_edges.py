"""MXFP4 operators on both sides of the rules that choose between their forms, and at values where they can go wrong.

The bounds are test_gpu_mx4.py's: quantised values are exact, a product's error is bounded by its number of f32
additions, the expert layer's by what those errors can do to its quantised activations."""

from __future__ import annotations

import pytest
import torch

from test_gpu_mx4 import check_product, experts_case, experts_reference, mx4_values, quantize, run_experts
from test_gpu_permute import UNIT

pytestmark = pytest.mark.gpu


# tokens of K summed values: at most 320 blocks are quantised by the product itself, more by a launch of their own
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("T,N,K", [(14, 300, 704), (15, 300, 704), (10, 129, 1024), (11, 129, 1024), (1, 200, 8192),
                                   (2, 200, 8192), (5, 130, 2048), (6, 130, 2048), (16, 257, 640), (16, 257, 641)])
def test_linear_on_both_sides_of_its_rule(cuda, moe, T, N, K, dtype):
    g = torch.Generator(device=cuda).manual_seed(T * K)
    x, w = torch.randn(T, K, generator=g, device=cuda).to(dtype), torch.randn(N, K, generator=g, device=cuda).to(dtype)
    out, ws = torch.full((T, N), 3.0, dtype=dtype, device=cuda), moe.new_mx4_linear_workspace(T, N, K, cuda)
    moe.mx4_linear(x, quantize(moe, w), out, T, N, K, ws)
    assert moe.device_status(ws)[0] == 0
    check_product(out, mx4_values(x), mx4_values(w), dtype)


# few pairs: 16 tokens, 128 pairs and 2048 blocks are the most that take three launches
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("T,K,E,H,I", [(8, 8, 16, 8192, 33), (9, 8, 16, 8192, 33), (16, 8, 64, 4096, 40), (16, 2, 8, 4160, 40),
                                       (16, 8, 8, 96, 64), (16, 9, 16, 96, 64), (2, 64, 128, 320, 33)])
def test_layer_on_both_sides_of_its_rule(cuda, moe, T, K, E, H, I, dtype):
    c = experts_case(T * K, T, K, E, H, I, dtype, cuda, 0.1)
    out, ws = run_experts(moe, c, T, K, E, H, I)
    assert moe.device_status(ws)[0] == 0
    want, tol = experts_reference(c, T, K, E, H, I)
    assert ((out.double() - want).abs() <= tol).all()


# from 80 million gathered values, and with more than one slot, the tokens are quantised before they are gathered
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("T,K,E,H,I,drop", [(10000, 8, 16, 1001, 40, 0.1), (9980, 8, 16, 1001, 40, 0.0), (6700, 12, 24, 1001, 33, 0.3),
                                            (20100, 4, 9, 1000, 40, 0.0), (80100, 1, 5, 1000, 33, 0.1), (1300, 8, 8, 8192, 33, 0.05)])
def test_large_layer_on_both_sides_of_its_rule(cuda, moe, T, K, E, H, I, drop, dtype):
    c = experts_case(T + K, T, K, E, H, I, dtype, cuda, drop)
    out, ws = run_experts(moe, c, T, K, E, H, I)
    assert moe.device_status(ws)[0] == 0
    want, tol = experts_reference(c, T, K, E, H, I)
    assert ((out.double() - want).abs() <= tol).all()
    again, _ = run_experts(moe, c, T, K, E, H, I, ws=ws)
    assert torch.equal(again, out)


def test_a_layer_workspace_serves_fewer_tokens(moe):
    """Also where the two-step gather begins, which depends on the tokens' width."""
    lib = moe.load_library()
    for H, K in ((256, 8), (1001, 8), (2816, 8), (8192, 2), (8192, 1)):
        at = 80_000_000 // (H * K)
        sizes = [lib.mrml_moe_mx4_experts_workspace_bytes(H, 64, 16, K, T) for T in range(at - 20, at + 20)]
        assert sizes == sorted(sizes)
