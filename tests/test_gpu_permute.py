"""Tokens sorted by expert and back (mrml_moe_sort, _permute, _unpermute) and
their gradients, against 64-bit restatements.

Tolerances, with u the unit roundoff of the row type (2^-24, 2^-11, 2^-8):
a sum of K products in f32 errs by at most (K + 1) 2^-24 of the sum of their
magnitudes, a dot of H products by (H + 1) 2^-24 of theirs, and the result is
then rounded once (u of its magnitude; f16's and bf16's subnormals are below
2^-24 and 2^-126).  Sorting and gathering are exact.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
F32 = 2.0**-24


def routing(seed, T, K, E, drop=0.0, one=None):
    rng = np.random.Generator(np.random.PCG64(seed))
    if one is not None:
        ids = np.full((T, K), one, np.int32)
    else:
        ids = np.argsort(rng.random((T, E)) + 0.5 * np.linspace(0, 1, E), axis=1)[:, :K].astype(np.int32) \
            if K <= E else rng.integers(0, E, (T, K)).astype(np.int32)
    ids[rng.random((T, K)) < drop] = -1
    return ids


def sort_numpy(ids, E, align, n_rows):
    flat = ids.reshape(-1)
    counts = np.array([(flat == e).sum() for e in range(E)], np.int64)
    offsets = np.concatenate([[0], np.cumsum((counts + align - 1) // align * align)])
    pos = np.full(flat.size, -1, np.int64)
    pair = np.full(n_rows, -1, np.int64)
    for e in range(E):
        p = np.nonzero(flat == e)[0]
        pos[p] = offsets[e] + np.arange(p.size)
        pair[pos[p]] = p
    return offsets, counts, pos.reshape(ids.shape), pair


def run_sort(moe, cuda, ids, E, align, ws=None):
    T, K = ids.shape
    n = moe.sorted_rows(E, K, T, align)
    i32 = dict(dtype=torch.int32, device=cuda)
    out = [torch.full((E + 1,), 77, **i32), torch.full((E,), 77, **i32), torch.full((T, K), 77, **i32),
           torch.full((n,), 77, **i32)]
    ws = moe.new_sort_workspace(E, K, T, cuda) if ws is None else ws
    moe.sort(torch.from_numpy(ids).to(cuda), *out, E, K, T, align, ws)
    return out, ws


SORTS = [
    (0, 8, 128, 1, 0.0, None), (1, 1, 1, 1, 0.0, None), (1, 8, 128, 128, 0.0, None), (3, 2, 5, 7, 0.5, None),
    (33, 8, 128, 1, 0.1, None), (64, 8, 256, 16, 0.0, None), (129, 64, 64, 128, 0.0, None), (511, 2, 16, 1, 1.0, None),
    (512, 8, 128, 8, 0.0, 127), (513, 8, 128, 1, 0.02, None), (2048, 2, 16, 128, 0.0, 3), (9001, 8, 61, 32, 0.3, None),
    (70000, 8, 256, 1, 0.01, None),
]


@pytest.mark.parametrize("T,K,E,align,drop,one", SORTS)
def test_sort(cuda, moe, T, K, E, align, drop, one):
    ids = routing(T + K, T, K, E, drop, one)
    (offsets, counts, pos, pair), ws = run_sort(moe, cuda, ids, E, align)
    ref = sort_numpy(ids, E, align, pair.numel())
    for got, want in zip((offsets, counts, pos, pair), ref):
        assert np.array_equal(got.cpu().numpy(), want)
    assert moe.device_status(ws)[0] == 0
    # the same again, in the same workspace
    again, _ = run_sort(moe, cuda, ids, E, align, ws)
    assert all(torch.equal(a, b) for a, b in zip(again, (offsets, counts, pos, pair)))


@pytest.mark.parametrize("T", [5, 3000])
def test_sort_skips_and_reports_ids_past_the_experts(cuda, moe, T):
    E, K = 16, 2
    ids = routing(1, T, K, E)
    bad = ids.copy()
    bad[T // 2, 1] = E
    bad[T - 1, 0] = 2**31 - 1
    (offsets, counts, pos, pair), ws = run_sort(moe, cuda, bad, E, 1)
    assert moe.device_status(ws)[0] == -7
    ref = sort_numpy(bad, E, 1, pair.numel())
    for got, want in zip((offsets, counts, pos, pair), ref):
        assert np.array_equal(got.cpu().numpy(), want)
    run_sort(moe, cuda, ids, E, 1, ws)
    assert moe.device_status(ws)[0] == 0


def strided(T, H, dtype, device, pad, shift, fill=None):
    """A [T][H] view with row stride H + pad that starts `shift` elements into its buffer."""
    buf = torch.full((T * (H + pad) + shift + 8,), 0.0 if fill is None else fill, dtype=dtype, device=device)
    return buf, buf[shift:shift + T * (H + pad)].view(T, H + pad)[:, :H]


# T, K, E, H, row stride - H, first element, dropped
SHAPES = [
    (1, 1, 1, 1, 0, 0, 0.0), (1, 8, 128, 2816, 0, 0, 0.0), (7, 2, 16, 33, 0, 0, 0.2), (64, 8, 128, 512, 8, 0, 0.0),
    (64, 3, 16, 1001, 3, 1, 0.5), (65, 8, 61, 1024, 0, 1, 0.0), (130, 64, 64, 40, 24, 8, 0.3), (9, 4, 8, 264, 0, 0, 1.0),
    (600, 8, 128, 2816, 0, 0, 0.05),
]


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("T,K,E,H,pad,shift,drop", SHAPES)
def test_rows_there_and_back(cuda, moe, T, K, E, H, pad, shift, drop, dtype):
    g = torch.Generator(device=cuda).manual_seed(T * 1000 + H)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    ids = routing(T + H, T, K, E, drop)
    align = 1 if T % 2 else 16
    (offsets, counts, pos, pair), _ = run_sort(moe, cuda, ids, E, align)
    n = pair.numel()
    u = UNIT[dtype]
    _, x = strided(T, H, dtype, cuda, pad, shift)
    x.copy_(rnd(T, H))
    probs = torch.rand(T, K, generator=g, device=cuda)
    tok = (pair.long().clamp(min=0) // K)
    used = (pair >= 0)[:, None]

    rows = torch.full((n, H), 9.0, dtype=dtype, device=cuda)
    moe.permute(x, pair, rows, H, K)
    assert torch.equal(rows, torch.where(used, x[tok], torch.zeros((), dtype=dtype, device=cuda)))

    y = rnd(n, H).to(dtype)
    has = (pos >= 0)[..., None]
    at = y[pos.long().clamp(min=0)].double() * has  # [T][K][H]

    def close(got, terms):
        want, mag = terms.sum(1), terms.abs().sum(1)
        tol = (K + 1) * F32 * mag + u * (want.abs() + (K + 1) * F32 * mag) + 2.0**-24 * (dtype == torch.float16)
        assert ((got.double() - want).abs() <= tol).all()

    obuf, out = strided(T, H, dtype, cuda, pad, shift, fill=5.0)
    moe.unpermute(y, pos, probs, out, H, K, T)
    close(out, at * probs.double()[..., None])
    edge = torch.ones_like(obuf, dtype=torch.bool)
    edge[shift:shift + T * (H + pad)].view(T, H + pad)[:, :H] = False
    assert (obuf[edge] == 5.0).all(), "written outside the output"

    _, dx = strided(T, H, dtype, cuda, pad, shift)
    moe.permute_grad(y, pos, dx, H, K, T)
    close(dx, at)
    _, ones = strided(T, H, dtype, cuda, pad, shift)
    moe.unpermute(y, pos, None, ones, H, K, T)
    assert torch.equal(dx, ones)

    _, dout = strided(T, H, dtype, cuda, pad, shift)
    dout.copy_(rnd(T, H))
    drows = torch.full((n, H), 9.0, dtype=dtype, device=cuda)
    dprobs = torch.full((T, K), 9.0, device=cuda)
    moe.unpermute_grad(dout, y, pos, pair, probs, drows, dprobs, H, K, T)
    w = probs.reshape(-1)[pair.long().clamp(min=0)].double()[:, None]
    want = torch.where(used, w * dout[tok].double(), 0.0)
    tol = (u + F32) * want.abs() * (1 + 2.0**-8) + 2.0**-24 * (dtype == torch.float16)
    assert ((drows.double() - want).abs() <= tol).all()
    prod = at * dout.double()[:, None, :]
    assert ((dprobs.double() - prod.sum(-1)).abs() <= (H + 1) * F32 * prod.abs().sum(-1)).all()
    assert (dprobs[pos < 0] == 0).all()

    # either output alone
    only = torch.full_like(drows, 9.0)
    moe.unpermute_grad(dout, None, pos, pair, probs, only, None, H, K, T)
    assert torch.equal(only, drows)
    alone = torch.full_like(dprobs, 9.0)
    moe.unpermute_grad(dout, y, pos, pair, probs, None, alone, H, K, T)
    assert torch.equal(alone, dprobs)


def test_gradients_against_differences(cuda, moe):
    """unpermute(f(permute(x))) with f a fixed map of rows: the directional
    derivatives from the gradient kernels against central differences of the
    forward kernels.  The map is linear in x and bilinear in (rows, probs), so
    differences have no truncation error; with values of order 1 and a step of
    1/4, f32 rounding of the two losses (sums of T*H = 3150 terms in 64 bits,
    each off by at most a few 2^-24) stays below 1e-3 of a derivative's scale
    sqrt(T*H)."""
    T, K, E, H = 42, 4, 9, 75
    g = torch.Generator(device=cuda).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g, device=cuda)  # noqa: E731
    ids = routing(3, T, K, E, 0.15)
    (_, _, pos, pair), _ = run_sort(moe, cuda, ids, E, 1)
    n = pair.numel()
    x, probs, mix, c = rnd(T, H), torch.rand(T, K, generator=g, device=cuda), rnd(n, H), rnd(T, H)

    def forward(x, probs):
        rows, out = torch.empty(n, H, device=cuda), torch.empty(T, H, device=cuda)
        moe.permute(x.contiguous(), pair, rows, H, K)
        y = rows * mix
        moe.unpermute(y, pos, probs.contiguous(), out, H, K, T)
        return (out.double() * c.double()).sum().item(), y

    _, y = forward(x, probs)
    drows, dprobs, dx = torch.empty_like(y), torch.empty_like(probs), torch.empty_like(x)
    moe.unpermute_grad(c, y, pos, pair, probs, drows, dprobs, H, K, T)
    moe.permute_grad(drows * mix, pos, dx, H, K, T)
    h, scale = 0.25, (T * H) ** 0.5
    for _ in range(3):
        v, q = rnd(T, H), rnd(T, K)
        num = (forward(x + h * v, probs)[0] - forward(x - h * v, probs)[0]) / (2 * h)
        assert abs(num - (dx.double() * v.double()).sum().item()) <= 1e-3 * scale
        num = (forward(x, probs + h * q)[0] - forward(x, probs - h * q)[0]) / (2 * h)
        assert abs(num - (dprobs.double() * q.double()).sum().item()) <= 1e-3 * scale


def test_non_finite_rows_stay_with_their_tokens(cuda, moe):
    T, K, E, H = 20, 2, 4, 72
    ids = routing(8, T, K, E, 0.2)
    (_, _, pos, pair), _ = run_sort(moe, cuda, ids, E, 1)
    y = torch.ones(pair.numel(), H, device=cuda)
    hit = int(pos[3].max())
    assert hit >= 0
    y[hit, 5] = float("inf")
    y[hit, 6] = float("nan")
    out = torch.empty(T, H, device=cuda)
    moe.unpermute(y, pos, torch.ones(T, K, device=cuda), out, H, K, T)
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[3, 5:7] = True
    assert torch.equal(bad, want)


def test_side_stream_and_graph(cuda, moe):
    """The calls run on the stream they are given, and a captured step replays
    on new contents of the same buffers."""
    T, K, E, H = 50, 8, 128, 256
    s = torch.cuda.Stream()
    ids = torch.from_numpy(routing(1, T, K, E)).to(cuda)
    x = torch.randn(T, H, device=cuda)
    n = moe.sorted_rows(E, K, T)
    i32 = dict(dtype=torch.int32, device=cuda)
    offsets, counts = torch.empty(E + 1, **i32), torch.empty(E, **i32)
    pos, pair = torch.empty(T, K, **i32), torch.empty(n, **i32)
    rows, out = torch.empty(n, H, device=cuda), torch.empty(T, H, device=cuda)
    probs = torch.full((T, K), 1.0 / K, device=cuda)
    ws = moe.new_sort_workspace(E, K, T, cuda)

    def step(stream):
        moe.sort(ids, offsets, counts, pos, pair, E, K, T, 1, ws, stream=stream)
        moe.permute(x, pair, rows, H, K, stream=stream)
        moe.unpermute(rows, pos, probs, out, H, K, T, stream=stream)

    s.wait_stream(torch.cuda.current_stream())
    step(s)
    torch.cuda.synchronize()
    tol = 10 * F32 * x.abs()
    assert ((out - x).abs() <= tol).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step(s)
    x.copy_(torch.randn(T, H, device=cuda))
    ids.copy_(torch.from_numpy(routing(2, T, K, E)).to(cuda))
    graph.replay()
    torch.cuda.synchronize()
    assert ((out - x).abs() <= 10 * F32 * x.abs()).all()
    ref = sort_numpy(ids.cpu().numpy(), E, 1, n)
    assert np.array_equal(pair.cpu().numpy(), ref[3])


def test_offsets_past_32_bits(cuda, moe):
    """262144 rows of 8704 16-bit values: 2.28e9 elements, 4.6 GB on each side of the gather."""
    T, K, E, H = 65536, 4, 16, 8704
    ids = routing(11, T, K, E)
    (_, _, pos, pair), _ = run_sort(moe, cuda, ids, E, 1)
    x = torch.empty(T, H, dtype=torch.bfloat16, device=cuda).normal_(generator=torch.Generator(cuda).manual_seed(1))
    rows = torch.empty(T * K, H, dtype=torch.bfloat16, device=cuda)
    moe.permute(x, pair, rows, H, K)
    at = torch.cat([torch.arange(0, T * K, 977, device=cuda), torch.arange(T * K - 50, T * K, device=cuda)])
    assert torch.equal(rows[at], x[pair[at].long() // K])
    out = torch.empty_like(x)
    moe.unpermute(rows, pos, torch.full((T, K), 0.25, device=cuda), out, H, K, T)
    assert torch.equal(out, x)  # sums of quarters of one value are exact
    drows, dprobs = torch.empty_like(rows), torch.empty(T, K, device=cuda)
    moe.unpermute_grad(x, rows, pos, pair, torch.full((T, K), 0.5, device=cuda), drows, dprobs, H, K, T)
    assert torch.equal(drows[at], 0.5 * x[pair[at].long() // K])
    t = torch.tensor([0, 1, T // 2, T - 1], device=cuda)
    sq = x[t].double().square().sum(1)
    assert ((dprobs[t].double() - sq[:, None]).abs() <= (H + 1) * F32 * sq[:, None]).all()
