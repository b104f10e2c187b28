"""Edges of the permutation operators: buffers longer than the batch, views, empty batches, the calls that come right
before and after.  Sorting and gathering are exact, and the sums here have one term or none, so results are compared for
equality."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_permute import routing, run_sort, sort_numpy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("align", [1, 16])
@pytest.mark.parametrize("few", [0, 1, 5, 300])
def test_buffers_of_a_larger_batch_serve_a_smaller_one(cuda, moe, few, align):
    """A sort of many tokens, then one of few into the same buffers: no row of the first is left."""
    T, K, E, H = 600, 4, 16, 40
    (offsets, counts, pos, pair), ws = run_sort(moe, cuda, routing(1, T, K, E), E, align)
    assert (pair >= 0).sum() == T * K
    ids = routing(2, few, K, E, 0.2)
    pos = pos[:few]
    for stream in (None, torch.cuda.Stream()):
        pair.fill_(T * K - 1)
        torch.cuda.synchronize()
        moe.sort(torch.from_numpy(ids).to(cuda), offsets, counts, pos, pair, E, K, few, align, ws, stream=stream)
        torch.cuda.synchronize()
        assert np.array_equal(pair.cpu().numpy(), sort_numpy(ids, E, align, pair.numel())[3])
    x = torch.randn(few, H, device=cuda)
    rows = torch.full((pair.numel(), H), 9.0, device=cuda)
    if few:
        moe.permute(x, pair, rows, H, K)
        want = torch.where((pair >= 0)[:, None], x[pair.long().clamp(min=0) // K], 0.0)
        assert torch.equal(rows, want)
        drows, dprobs = torch.full_like(rows, 9.0), torch.empty(few, K, device=cuda)
        moe.unpermute_grad(x, rows, pos, pair, None, drows, dprobs, H, K, few)
        assert torch.equal(drows, want)


def test_views_with_more_axes(cuda, moe):
    """[batch][length][H] views: those whose rows lie at one stride are read as they are, others are refused."""
    B, L, K, E, H = 5, 9, 2, 8, 24
    base = torch.randn(B, L, 2 * H, device=cuda)
    views = {
        "whole": base, "columns": base[:, :, :H], "last": base[:, -1:, :], "one batch": base[1:2, 2:7, H:],
        "every second batch": base[::2, 3:4], "one row": base[3:4, 4:5, 3:], "flat": base[:, 2],
    }
    for name, x in views.items():
        T, h = x[..., 0].numel(), x.shape[-1]
        (_, _, _, pair), _ = run_sort(moe, cuda, routing(T, T, K, E), E, 1)
        rows = torch.full((pair.numel(), h), 9.0, device=cuda)
        moe.permute(x, pair, rows, h, K)
        assert torch.equal(rows, x.reshape(T, h)[pair.long() // K]), name
    for x in (base[:, :4], base[:, ::2], base.transpose(0, 1), base[:, :, ::2]):
        T, h = x[..., 0].numel(), x.shape[-1]
        (_, _, _, pair), _ = run_sort(moe, cuda, routing(T, T, K, E), E, 1)
        rows = torch.full((pair.numel(), h), 9.0, device=cuda)
        with pytest.raises(AssertionError):
            moe.permute(x, pair, rows, h, K)
        assert (rows == 9.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_an_empty_batch_clears_the_rows(cuda, moe, dtype):
    """No tokens, and a row buffer kept at its size: all its rows are without a pair, so their gradient is zero."""
    K, E, H, n = 2, 8, 33, 70
    i32 = dict(dtype=torch.int32, device=cuda)
    pos, pair = torch.empty(0, K, **i32), torch.full((n,), 3, **i32)
    ids, ws = torch.empty(0, K, **i32), moe.new_sort_workspace(E, K, 0, cuda)
    moe.sort(ids, torch.empty(E + 1, **i32), torch.empty(E, **i32), pos, pair, E, K, 0, 1, ws)
    assert (pair == -1).all()
    rows, buf = torch.ones(n, H, dtype=dtype, device=cuda), torch.full((n + 2, H), 5.0, dtype=dtype, device=cuda)
    drows, probs = buf[1:-1], torch.empty(0, K, device=cuda)
    moe.unpermute_grad(torch.empty(0, H, dtype=dtype, device=cuda), rows, pos, pair, probs, drows,
                       torch.empty(0, K, device=cuda), H, K, 0)
    assert (drows == 0).all() and (buf[0] == 5).all() and (buf[-1] == 5).all()
    # without a row gradient there is nothing to do
    moe.unpermute_grad(torch.empty(0, H, dtype=dtype, device=cuda), rows, pos, pair, probs, None,
                       torch.empty(0, K, device=cuda), H, K, 0)


@pytest.mark.parametrize("T", [1, 8])
def test_router_weights_written_right_before(cuda, moe, T):
    """Router weights that another operator of the library writes right before the router reads them, with fresh
    contents each time, in a stream and in a graph.  The logits are one fixed chain of additions, so they equal those of
    a settled copy."""
    H, E, K, rounds = 2816, 128, 8, 24
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(T, H, generator=g, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    ws, mm = moe.new_workspace(32, 32, E, K, T, cuda), moe.new_mx4_matmul_workspace(E, H, 64, cuda)
    W, codes = torch.zeros(E, H, device=cuda), moe.new_mx4(E, H, 1, cuda)
    a, b = moe.new_mx4(E, 64, 1, cuda), moe.new_mx4(H, 64, 1, cuda)
    moe.mx4_quantize(torch.randn(H, 64, generator=g, device=cuda), b, H, 64)
    order = torch.randperm(E, generator=g, device=cuda).to(torch.int32)
    base = torch.empty(E, H, device=cuda)

    def by_dequantising(new, s):
        moe.mx4_quantize(new, codes, E, H, stream=s)
        moe.mx4_dequantize(codes, W, E, H, stream=s)

    def by_product(new, s):
        moe.mx4_quantize(new[:, :64], a, E, 64, stream=s)
        moe.mx4_matmul(a, b, W, E, H, 64, mm, stream=s)

    def by_gathering(new, s):
        moe.permute(new, order, W, H, 1, stream=s)

    def by_summing(new, s):
        moe.unpermute(new, order, None, W, H, 1, E, stream=s)

    s = torch.cuda.Stream()
    for write in (by_dequantising, by_product, by_gathering, by_summing):
        logits, ids, probs = torch.empty(T, E, device=cuda), torch.empty(T, K, **i32), torch.empty(T, K, device=cuda)
        step = lambda: (write(base, s), moe.router(W, x, logits, ids, probs, H, E, K, T, ws, s))  # noqa: E731
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
        for i in range(rounds):
            base.normal_(generator=g)
            torch.cuda.synchronize()
            if i % 2:
                step()
            else:
                graph.replay()
            torch.cuda.synchronize()
            got = logits.clone(), ids.clone(), probs.clone()
            settled = W.clone()
            torch.cuda.synchronize()
            moe.router(settled, x, logits, ids, probs, H, E, K, T, ws)
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(got, (logits, ids, probs))), write.__name__


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_non_finite_values_stay_where_they_belong(cuda, moe, dtype):
    """Weights of dropped slots are not read as factors, and a token's non-finite values reach its own results only."""
    T, K, E, H = 30, 3, 5, 72
    ids = routing(4, T, K, E, 0.4)
    ids[7], ids[8, 0], ids[9, 1] = -1, 2, 3  # a token without any slot, and two that have one
    (_, _, pos, pair), _ = run_sort(moe, cuda, ids, E, 1)
    none = pos < 0
    probs = torch.rand(T, K, device=cuda).masked_fill(none, float("nan"))
    rows = torch.ones(pair.numel(), H, dtype=dtype, device=cuda)
    rows[(pair < 0)] = float("nan")
    out = torch.full((T, H), 9.0, dtype=dtype, device=cuda)
    moe.unpermute(rows, pos, probs, out, H, K, T)
    assert torch.isfinite(out).all() and (out[7] == 0).all()
    dout = torch.ones(T, H, dtype=dtype, device=cuda)
    dout[7, 1], dout[8, 5], dout[9, 6] = float("nan"), float("inf"), float("nan")
    drows, dprobs = torch.full_like(rows, 9.0), torch.full_like(probs, 9.0)
    moe.unpermute_grad(dout, rows, pos, pair, probs, drows, dprobs, H, K, T)
    token = torch.where(pair >= 0, pair // K, -1)
    bad = torch.zeros_like(rows, dtype=torch.bool)
    bad[token == 8, 5], bad[token == 9, 6] = True, True
    assert torch.equal(~torch.isfinite(drows), bad) and (drows[pair < 0] == 0).all()
    want = torch.zeros_like(none)
    want[8], want[9] = ~none[8], ~none[9]
    assert torch.equal(~torch.isfinite(dprobs), want) and (dprobs[none] == 0).all()
