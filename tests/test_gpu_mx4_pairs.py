"""Products by pairs of CTAs: what passes between the two CTAs, under repetition.

A product's result is a fixed sum of exact terms, so every repetition has to
give the same bits, whatever runs before, after or between.  The first result
of each shape is checked against 64 bits by test_gpu_mx4.py's bound.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_mx4 import check_product, mx4_values, quantize

pytestmark = pytest.mark.gpu

# M, N, K of paired products: short and ragged chunks, ragged token tiles, an odd number of weight tiles
PAIRED = [(4000, 3330, 1056), (9001, 1500, 1100), (4096, 4224, 1024)]


def product(moe, device, M, N, K, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    x, w = torch.randn(M, K, generator=g, device=device), torch.randn(N, K, generator=g, device=device)
    qx, qw = quantize(moe, x), quantize(moe, w)
    out = torch.zeros(M, N, dtype=torch.bfloat16, device=device)
    ws = moe.new_mx4_matmul_workspace(M, N, K, device)
    return (x, w), lambda stream=None: moe.mx4_matmul(qx, qw, out, M, N, K, ws, stream=stream), out, ws


@pytest.mark.parametrize("M,N,K", PAIRED)
def test_nothing_of_a_pair_outlives_it(cuda, moe, M, N, K):
    """Pairs and single CTAs follow one another without a gap, on the same SMs and with their barriers at the same
    places of shared memory: a signal of a pair that came after one of its CTAs had left would count for the next."""
    (x, w), big, out, ws = product(moe, cuda, M, N, K, 1)
    _, small, few, ws2 = product(moe, cuda, 3, 20000, 96, 2)
    big()
    small()
    check_product(out, mx4_values(x), mx4_values(w), torch.bfloat16)
    first, first_few = out.clone(), few.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        for _ in range(8):
            big(s)
            small(s)
            small(s)
    for _ in range(25):
        out.zero_()
        few.zero_()
        graph.replay()
        assert torch.equal(out, first) and torch.equal(few, first_few)
    assert moe.device_status(ws)[0] == 0 and moe.device_status(ws2)[0] == 0


@pytest.mark.parametrize("M,N,K", PAIRED)
def test_a_pair_reads_what_has_landed(cuda, moe, M, N, K):
    """Two products of one shape in turn, so that a stage read before its copy had landed in either CTA would hold the
    other product's operands (or another unit's)."""
    runs = [product(moe, cuda, M, N, K, seed) for seed in (3, 4)]
    first = []
    for (x, w), run, out, _ in runs:
        run()
        check_product(out, mx4_values(x), mx4_values(w), torch.bfloat16)
        first.append(out.clone())
    for _ in range(40):
        for _, run, out, _ in runs:
            run()
        assert all(torch.equal(r[2], f) for r, f in zip(runs, first))
    assert all(moe.device_status(r[3])[0] == 0 for r in runs)
