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
