"""MXFP4 operators on both sides of the rules that choose between their forms, and at values where they can go wrong.

The bounds are test_gpu_mx4.py's: quantised values are exact, a product's error is bounded by its number of f32
additions, the expert layer's by what those errors can do to its quantised activations."""

from __future__ import annotations

import pytest
import torch

from test_gpu_mx4 import (check_product, experts_case, experts_reference, mx4_values, quantize, run_experts, same,
                          values)
from test_gpu_permute import UNIT, strided

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


def special_rows(dtype, device):
    """Rows of 96 values: infinities and NaN of either sign in every part of a block, and the type's subnormals."""
    inf, nan = float("inf"), float("nan")
    tiny = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}[dtype]
    rows = [[tiny * (1 + (i * 37) % 120) * (-1) ** i for i in range(96)], [tiny] * 32 + [-tiny] * 32 + [0.0] * 32,
            [tiny * 64] * 16 + [-tiny * 127] * 16 + [0.0] * 64, [-0.0] * 96]
    for bad in (inf, -inf, nan, -nan):
        for at in (0, 1, 15, 16, 31, 32, 63, 64, 95):
            row = [0.5 * (i % 7) - 1 for i in range(96)]
            row[at] = bad
            rows.append(row)
    rows.append([torch.finfo(dtype).max * (-1) ** i for i in range(96)])
    rows.append([1.0] * 95 + [inf])
    rows.append([nan, inf] + [0.0] * 94)
    return torch.tensor(rows, dtype=torch.float64, device=device).to(dtype)


@pytest.mark.parametrize("dtype", list(UNIT))
def test_special_values_of_every_type(cuda, moe, dtype):
    x = special_rows(dtype, cuda)
    n, c = x.shape
    want = mx4_values(x)
    assert torch.isnan(want).any() and torch.isfinite(want[:4]).all()
    # vectors, and element by element (unaligned rows)
    for pad, shift in ((0, 0), (8, 0), (3, 1)):
        _, v = strided(n, c, dtype, cuda, pad, shift)
        v.copy_(x)
        q, qt = moe.new_mx4(n, c, 1, cuda), moe.new_mx4(c, n, 1, cuda)
        assert same(values(moe, quantize(moe, v), n, c)[0], want)
        moe.mx4_quantize_both(v, q, qt, n, c)
        assert same(values(moe, q, n, c)[0], want)
        assert same(values(moe, qt, c, n)[0], mx4_values(x.t()))


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("T,K", [(3, 2), (16, 8), (40, 4), (10100, 8)])
def test_special_tokens_stay_apart_in_every_type(cuda, moe, T, K, dtype):
    """In each of the layer's forms (sorted in the product, gathered in one and in two steps), and in the linear layer."""
    E, H, I = 8, 1000, 40
    c = experts_case(T, T, K, E, H, I, dtype, cuda)
    clean, _ = run_experts(moe, c, T, K, E, H, I)
    c["x"] = c["x"].clone()
    bad = torch.zeros(T, dtype=torch.bool, device=cuda)
    for t, at, v in ((0, 0, "inf"), (1, 999, "nan"), (T - 1, 517, "-inf")):
        c["x"][t, at] = float(v)
        bad[t] = True
    out, _ = run_experts(moe, c, T, K, E, H, I)
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
    w = quantize(moe, c["down"][0])  # [H][I]
    x = c["x"][:, :I].contiguous()
    y, ws = torch.empty(T, H, dtype=dtype, device=cuda), moe.new_mx4_linear_workspace(T, H, I, cuda)
    moe.mx4_linear(x, w, y, T, H, I, ws)
    bad[:] = False
    bad[0] = True  # the one whose mark lies in the first I columns
    assert torch.isnan(y[bad]).all() and torch.isfinite(y[~bad]).all()


@pytest.mark.parametrize("dtype", list(UNIT))
def test_layer_of_subnormal_tokens(cuda, moe, dtype):
    T, K, E, H, I = 20, 2, 4, 96, 64
    c = experts_case(3, T, K, E, H, I, dtype, cuda)
    c["x"] = special_rows(dtype, cuda)[:4].repeat(5, 1)
    c["gate_up"] = (c["gate_up"].float() * 2.0**12).to(dtype)
    out, _ = run_experts(moe, c, T, K, E, H, I)
    want, tol = experts_reference(c, T, K, E, H, I)
    assert ((out.double() - want).abs() <= tol).all()


# ------------------------------------------------------------ streams and threads


def layer_steps(moe, device, seed):
    """Calls of every form, with buffers of their own, and their first results."""
    steps = []
    for T, K, E, H, I in ((4, 8, 16, 1000, 96), (100, 4, 8, 520, 200), (3000, 8, 7, 1040, 333)):
        c = experts_case(seed + T, T, K, E, H, I, torch.bfloat16, device)
        qg, qd = quantize(moe, c["gate_up"], gated=True), quantize(moe, c["down"])
        out, ws = torch.empty_like(c["x"]), moe.new_mx4_experts_workspace(H, I, E, K, T, device)

        def step(stream=None, a=(qg, qd, c["ids"], c["probs"], c["scale"], c["x"], out, H, I, E, K, T, ws)):
            moe.mx4_experts(*a, stream=stream)

        steps.append((step, out, ws))
    for step, _, _ in steps:
        step()
    torch.cuda.synchronize()
    return steps, [o.clone() for _, o, _ in steps]


def test_two_streams(cuda, moe):
    """Calls on two streams at once, each with its own workspaces: what each gives alone."""
    sides = [layer_steps(moe, cuda, seed) for seed in (1, 2)]
    streams = [torch.cuda.Stream() for _ in sides]
    torch.cuda.synchronize()
    for _ in range(30):
        for j in range(3):
            for (steps, _), s in zip(sides, streams):
                steps[j][0](s)
    torch.cuda.synchronize()
    for steps, first in sides:
        assert all(torch.equal(o, f) and moe.device_status(ws)[0] == 0 for (_, o, ws), f in zip(steps, first))


def test_two_threads(cuda, moe):
    """The same from two host threads, each on a stream of its own."""
    import threading

    sides = [layer_steps(moe, cuda, seed) for seed in (3, 4)]
    torch.cuda.synchronize()
    errors = []

    def work(steps):
        try:
            s = torch.cuda.Stream()
            for _ in range(40):
                for step, _, _ in steps:
                    step(s)
            s.synchronize()
        except Exception as e:  # noqa: BLE001 (a thread's exception would be lost)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(steps,)) for steps, _ in sides]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for steps, first in sides:
        assert all(torch.equal(o, f) and moe.device_status(ws)[0] == 0 for (_, o, ws), f in zip(steps, first))
