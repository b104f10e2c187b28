"""MXFP4: quantisation, products and the expert layer, against 64-bit
restatements of the format and of the formulas.

Quantised values are exact (every rounding is defined), so they are compared
for equality.  A product's terms are exact; the tensor cores add them in f32,
64 at a time: with at most one truncating f32 addition per 64 terms and one
more inside, a sum of S such steps errs by at most (S + 2) 2^-23 of the sum of
magnitudes, and is then rounded once to the output type.  The expert layer's
tolerance is derived in its test.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_permute import UNIT, routing, strided

pytestmark = pytest.mark.gpu

TABLE = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# midpoints between neighbours, and whether a tie goes to the larger one
MIDS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))


def pow2(e):
    """2^e in 64 bits, from its bits (torch.pow is not exact on the GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def blocks_of(x):
    x = x.double()
    pad = -x.shape[-1] % 32
    return torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, 32))


def scale_exponents(b):
    """floor(log2(max)) - 2 of finite blocks, at least -127, from the doubles' bits."""
    big = b.abs().amax(-1, keepdim=True)
    return ((big.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127)


def mx4_codes(x):
    """(codes 0..15, scale bytes) of a matrix' blocks: [.., block, 32], [.., block]."""
    b = blocks_of(x)
    finite = torch.isfinite(b).all(-1, keepdim=True)
    e = scale_exponents(torch.where(finite, b, 0.0))
    a = b.abs() * pow2(-e)
    code = sum(((a >= m) if up else (a > m)).long() for m, up in MIDS)
    code = code + 8 * torch.signbit(b).long()
    return code, torch.where(finite, e + 127, 255)[..., 0]


def mx4_values(x):
    code, s = mx4_codes(x)
    v = TABLE.to(x.device)[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    v = v * pow2(s - 127)[..., None]
    v = torch.where((s == 255)[..., None], float("nan"), v)
    return v.flatten(-2)[..., :x.shape[-1]]


def same(a, b):
    """Equal as numbers, NaN in the same places."""
    a, b = a.double(), b.double()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


def quantize(moe, x, gated=False):
    m = x if x.dim() == 3 else x[None]
    n, r, c = m.shape
    q = moe.new_mx4(r, c, n, x.device)
    q.fill_(0xA5)
    moe.mx4_quantize(x, q, r, c, n, gated=gated)
    return q


def values(moe, q, rows, cols, n=1, gated=False, dtype=torch.float32):
    out = torch.full((n, rows, cols), 3.0, dtype=dtype, device=q.device)
    moe.mx4_dequantize(q, out, rows, cols, n, gated=gated)
    return out


SHAPES = [(1, 1), (1, 32), (3, 33), (16, 64), (127, 31), (128, 256), (129, 257), (33, 1000), (300, 2816), (257, 704)]


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantised_values(cuda, moe, rows, cols, dtype):
    g = torch.Generator(device=cuda).manual_seed(rows * 7 + cols)
    x = torch.randn(rows, cols, generator=g, device=cuda)
    x = (x * torch.exp(2 * torch.randn(rows, 1, generator=g, device=cuda))).to(dtype)
    q = quantize(moe, x)
    want = mx4_values(x)
    assert same(values(moe, q, rows, cols)[0], want)
    assert same(values(moe, q, rows, cols, dtype=torch.bfloat16)[0], want)
    half = values(moe, q, rows, cols, dtype=torch.float16)[0]
    assert same(half, want.half())
    # both directions in one read
    qr, qc = moe.new_mx4(rows, cols, 1, cuda), moe.new_mx4(cols, rows, 1, cuda)
    qr.fill_(0x5A)
    qc.fill_(0x5A)
    moe.mx4_quantize_both(x, qr, qc, rows, cols)
    assert torch.equal(written(qr, rows, cols), written(q, rows, cols))
    assert torch.equal(written(qc, cols, rows), written(quantize(moe, x.t().contiguous()), cols, rows))
    # strided input, unaligned input
    for pad, shift in ((8, 0), (3, 1)):
        _, v = strided(rows, cols, dtype, cuda, pad, shift)
        v.copy_(x)
        assert torch.equal(written(quantize(moe, v), rows, cols), written(q, rows, cols))
        moe.mx4_quantize_both(v, qr, qc, rows, cols)
        assert torch.equal(written(qr, rows, cols), written(q, rows, cols))
    # strided output
    buf, o = strided(rows, cols, torch.float32, cuda, 5, 3, fill=2.5)
    moe.mx4_dequantize(q, o, rows, cols)
    assert same(o, want)
    o.fill_(2.5)
    assert (buf == 2.5).all()


def layout(rows, cols):
    """Byte offsets of the layout, restated: codes [row][block][16], scales [row][block]."""
    nb = ((cols + 31) // 32 + 1) // 2 * 2
    chunk = 8 * 2048 + 1024
    n_last = nb % 8
    tile = nb // 8 * chunk + (n_last * 2048 + (n_last + 3) // 4 * 512 if n_last else 0)
    r = np.arange((rows + 127) // 128 * 128)[:, None]
    b = np.arange(nb)[None, :]
    c, bl = b // 8, b % 8
    n = np.minimum(8, nb - 8 * c)
    t, i = r // 128, r % 128
    base = t * tile + c * chunk
    code = base + (n + 3) // 4 * 512 + i // 8 * (n * 128) + bl * 128 + i % 8 * 16
    scale = base + bl // 4 * 512 + i % 32 * 16 + i // 32 * 4 + bl % 4
    return code, scale, nb, (rows + 127) // 128 * tile


def written(q, rows, cols):
    """The bytes of a matrix that the layout defines (a short chunk's scale groups have unused bytes)."""
    code, scale, _, size = layout(rows, cols)
    assert q.numel() == size
    at = np.concatenate([(code[..., None] + np.arange(16)).reshape(-1), scale.reshape(-1)])
    return q[torch.from_numpy(at).to(q.device)]


@pytest.mark.parametrize("rows,cols", [(1, 1), (130, 300), (128, 704), (40, 96)])
def test_layout(cuda, moe, rows, cols):
    """Codes and scales lie where the format says; rows and blocks past the matrix are zero."""
    x = torch.randn(rows, cols, device=cuda)
    q = quantize(moe, x).cpu().numpy()
    code, scale, nb, _ = layout(rows, cols)
    want, s = mx4_codes(x.cpu())
    full = np.zeros((code.shape[0], nb, 32), np.int64)
    fs = np.zeros((code.shape[0], nb), np.int64)
    full[:rows, :want.shape[1]] = want.numpy()
    fs[:rows, :s.shape[1]] = s.numpy()
    got = q[code[..., None] + np.arange(16)]
    lo, hi = got & 15, got >> 4
    zero = lambda c: np.where((c & 7) == 0, 0, c)  # noqa: E731 (either sign of zero)
    assert np.array_equal(zero(lo), zero(full[..., 0::2])) and np.array_equal(zero(hi), zero(full[..., 1::2]))
    assert np.array_equal(q[scale], fs)


def test_ties_saturation_and_special_values(cuda, moe):
    rows = []
    for e in (-126, -20, 0, 7, 120):
        mids = [m for m, _ in MIDS]
        near = [math.ldexp(v, e) for m in mids for v in (m, -m, m * (1 + 2**-20), -m * (1 - 2**-20))]
        rows.append([math.ldexp(4.0, e)] + near + [0.0, -0.0, math.ldexp(7.999, e)])
        rows.append([math.ldexp(7.9999, e), math.ldexp(6.5, e), -math.ldexp(7.0, e)] + [math.ldexp(0.24, e)] * 29)
    rows.append([0.0] * 32)
    rows.append([2.0**-149] * 16 + [2.0**-130] * 16)
    rows.append([3.4e38, -1.0e38] + [1.0] * 30)
    rows.append([1.0] * 31 + [float("inf")])
    rows.append([float("nan")] + [1.0] * 31)
    rows.append([1.0] * 32)
    x = torch.tensor(rows, dtype=torch.float64, device=cuda).float()
    q = quantize(moe, x)
    got, want = values(moe, q, len(rows), 32)[0], mx4_values(x)
    assert same(got, want)
    assert torch.isnan(got[-3:-1]).all() and torch.isfinite(got[-1]).all()
    qr, qt = moe.new_mx4(len(rows), 32, 1, cuda), moe.new_mx4(32, len(rows), 1, cuda)
    moe.mx4_quantize_both(x, qr, qt, len(rows), 32)
    assert same(values(moe, qr, len(rows), 32)[0], want)
    assert same(values(moe, qt, 32, len(rows))[0], mx4_values(x.t()))


@pytest.mark.parametrize("I,cols,n", [(64, 256, 2), (96, 100, 3), (1, 32, 1), (500, 1000, 2), (704, 2816, 2)])
def test_gated_matrices(cuda, moe, I, cols, n):
    x = torch.randn(n, 2 * I, cols, device=cuda).bfloat16()
    q = quantize(moe, x, gated=True)
    assert same(values(moe, q, 2 * I, cols, n, gated=True), mx4_values(x))


@pytest.mark.parametrize("wtype", [2, 8])
def test_gguf_blocks_as_source(cuda, moe, synth, oracle, wtype):
    E, rows, cols = 2, 192, 416
    w = synth.normal(3, E * rows * cols, 0.02).reshape(E, rows, cols)
    raw = (synth.quantize_q4_0 if wtype == 2 else synth.quantize_q8_0)(w)
    deq = np.stack([oracle.dequantize(raw[e].reshape(-1), wtype).reshape(rows, cols) for e in range(E)])
    src = torch.from_numpy(raw).to(cuda)
    for gated in (False, True):
        q = moe.new_mx4(rows, cols, E, cuda)
        moe.mx4_quantize(src, q, rows, cols, E, gated=gated, wtype=wtype)
        assert same(values(moe, q, rows, cols, E, gated=gated), mx4_values(torch.from_numpy(deq).to(cuda)))


# ----------------------------------------------------------------- products


def matmul(moe, x, w, dtype, out=None):
    (M, K), N = x.shape, w.shape[0]
    qx, qw = quantize(moe, x), quantize(moe, w)
    out = torch.full((M, N), 3.0, dtype=dtype, device=x.device) if out is None else out
    ws = moe.new_mx4_matmul_workspace(M, N, K, x.device)
    moe.mx4_matmul(qx, qw, out, M, N, K, ws)
    assert moe.device_status(ws)[0] == 0
    return out


def check_product(got, a, b, dtype):
    """got against a b^T of exact values."""
    steps = -(-a.shape[1] // 64)
    for r in range(0, a.shape[0], 8192):
        x, y = a[r:r + 8192], got[r:r + 8192]
        want, mag = x @ b.t(), x.abs() @ b.abs().t()
        tol = (steps + 2) * 2.0**-23 * mag
        tol = tol + UNIT[dtype] * (want.abs() + tol) + 2.0**-24 * (dtype == torch.float16)
        assert ((y.double() - want).abs() <= tol).all()


PRODUCTS = [
    (1, 1, 1), (1, 128, 64), (1, 129, 96), (5, 300, 2816), (16, 64, 32), (17, 257, 300), (128, 128, 256), (129, 130, 704),
    (100, 1000, 1000), (300, 704, 2816), (1, 2816, 4224), (513, 384, 640),
    # large ones are shared by pairs of CTAs: whole and ragged token tiles of 192, odd numbers of weight tiles, short
    # chunks of every length
    (192, 128, 64), (193, 129, 96), (384, 640, 320), (400, 257, 448), (575, 300, 1000), (1000, 130, 704), (2000, 900, 512),
    (4000, 3330, 1056), (9001, 1500, 1100), (12300, 1000, 1216), (100000, 130, 1024),
    # a few tokens, quantised by the product itself, up to and past its longest sum
    (2, 300, 33), (7, 129, 448), (8, 64, 704), (9, 1000, 96), (15, 260, 1000), (16, 4224, 2816), (3, 130, 8192),
    (2, 64, 8200), (1, 20000, 64),
]


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(cuda, moe, M, N, K, dtype):
    g = torch.Generator(device=cuda).manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g, device=cuda) * torch.exp(torch.randn(M, K, generator=g, device=cuda))
    w = torch.randn(N, K, generator=g, device=cuda) * 0.02
    x, w = x.to(dtype), w.to(dtype)
    a, b = mx4_values(x), mx4_values(w)
    check_product(matmul(moe, x, w, dtype), a, b, dtype)
    # through the linear layer, into a strided output
    buf, out = strided(M, N, dtype, cuda, 3, 1, fill=7.0)
    qw = quantize(moe, w)
    ws = moe.new_mx4_linear_workspace(M, N, K, cuda)
    moe.mx4_linear(x, qw, out, M, N, K, ws)
    assert moe.device_status(ws)[0] == 0
    check_product(out, a, b, dtype)
    # unaligned rows of x give the same
    _, xs = strided(M, K, dtype, cuda, 5, 1)
    xs.copy_(x)
    again = torch.full((M, N), 7.0, dtype=dtype, device=cuda)
    moe.mx4_linear(xs, qw, again, M, N, K, ws)
    assert torch.equal(again, out)
    out.fill_(7.0)
    assert (buf == 7.0).all(), "written outside the output"


def test_product_of_wide_scales_and_special_blocks(cuda, moe):
    """Scales from 2^-60 to 2^60 in one row; a NaN block reaches exactly the results of its row."""
    M, N, K = 20, 140, 320
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(M, K, generator=g, device=cuda)
    e = torch.randint(-60, 61, (M, K // 32), generator=g, device=cuda).repeat_interleave(32, 1)
    x = torch.ldexp(x, e)
    w = torch.randn(N, K, generator=g, device=cuda)
    check_product(matmul(moe, x, w, torch.float32), mx4_values(x), mx4_values(w), torch.float32)
    x[7, 100] = float("inf")
    w[130, 3] = float("nan")
    got = matmul(moe, x, w, torch.float32)
    bad = torch.zeros(M, N, dtype=torch.bool, device=cuda)
    bad[7], bad[:, 130] = True, True
    assert torch.equal(torch.isnan(got), bad)


def test_product_offsets_past_32_bits(cuda, moe):
    """70000 x 32768 results (2.3e9 elements), and 2.2e9 quantised values."""
    M, N, K = 70000, 32768, 64
    g = torch.Generator(device=cuda).manual_seed(6)
    x, w = torch.randn(M, K, generator=g, device=cuda), torch.randn(N, K, generator=g, device=cuda)
    out = matmul(moe, x, w, torch.bfloat16)
    at = torch.cat([torch.arange(0, M, 4999, device=cuda), torch.arange(M - 20, M, device=cuda)])
    check_product(out[at], mx4_values(x[at]), mx4_values(w), torch.bfloat16)
    q = quantize(moe, out)
    back = values(moe, q, M, N, dtype=torch.bfloat16)[0]
    assert same(back[at], mx4_values(out[at]))


def test_training_step_products(cuda, moe):
    """y = x w^T, dx = dy w and dw = dy^T x from three pairs of quantisations."""
    T, N, K = 200, 328, 264
    g = torch.Generator(device=cuda).manual_seed(4)
    x, w, dy = (torch.randn(*s, generator=g, device=cuda).bfloat16() for s in ((T, K), (N, K), (T, N)))
    q = {}
    for n, t in (("x", x), ("w", w), ("dy", dy)):
        r, c = t.shape
        q[n], q[n + "t"] = moe.new_mx4(r, c, 1, cuda), moe.new_mx4(c, r, 1, cuda)
        moe.mx4_quantize_both(t, q[n], q[n + "t"], r, c)
    v = lambda t: mx4_values(t)  # noqa: E731
    for a, b, M, n, k, ea, eb in (("x", "w", T, N, K, x, w), ("dy", "wt", T, K, N, dy, w.t()),
                                  ("dyt", "xt", N, K, T, dy.t(), x.t())):
        out = torch.empty(M, n, device=cuda)
        ws = moe.new_mx4_matmul_workspace(M, n, k, cuda)
        moe.mx4_matmul(q[a], q[b], out, M, n, k, ws)
        check_product(out, v(ea), v(eb), torch.float32)


# -------------------------------------------------------------- expert layer


def experts_case(seed, T, K, E, H, I, dtype, device, drop=0.0, one=None):
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    return dict(ids=torch.from_numpy(routing(seed, T, K, E, drop, one)).to(device),
                probs=torch.softmax(rnd(T, K), 1), scale=torch.rand(E, generator=g, device=device) + 0.5,
                x=rnd(T, H).to(dtype), gate_up=(0.05 * rnd(E, 2 * I, H)).to(dtype),
                down=(0.05 * rnd(E, H, I)).to(dtype))


def run_experts(moe, c, T, K, E, H, I, scaled=True, out=None, ws=None, stream=None):
    qg, qd = quantize(moe, c["gate_up"], gated=True), quantize(moe, c["down"])
    out = torch.full_like(c["x"], 3.0) if out is None else out
    ws = moe.new_mx4_experts_workspace(H, I, E, K, T, out.device) if ws is None else ws
    moe.mx4_experts(qg, qd, c["ids"], c["probs"], c["scale"] if scaled else None, c["x"], out, H, I, E, K, T, ws)
    return out, ws


def experts_reference(c, T, K, E, H, I, scaled=True):
    """(out, tol) in 64 bits.

    The activation a = gelu(g) u is computed in f32 before it is quantised.
    Its error d: g and u are off by at most (S + 2) 2^-23 of their terms'
    magnitudes; |gelu'| < 1.13; and the epilogue's own arithmetic (a product
    chain of 5 roundings, an exponential good to a few units plus the rounding
    of its argument z, one fast division) costs at most (12 + 4 |z|) 2^-23 |a|.
    Where a / scale lies within d of a midpoint the code may differ by one step
    (at most 2 scales), where the block's maximum lies within d of a power of
    two the whole block may be scaled otherwise (at most 4 scales per value);
    those differences times |down| and the routing weight, plus the rounding of
    the two sums and of the result, bound the output's error."""
    x = mx4_values(c["x"])
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    tol, mag = torch.zeros_like(out), torch.zeros_like(out)
    ids = c["ids"].long()
    for e in range(E):
        t, k = torch.nonzero(ids == e, as_tuple=True)
        if not len(t):
            continue
        w, dn = mx4_values(c["gate_up"][e]), mx4_values(c["down"][e])
        h, hm = x[t] @ w.t(), x[t].abs() @ w.abs().t()
        dh = (-(-H // 64) + 2) * 2.0**-23 * hm
        g, u, dg, du = h[:, :I], h[:, I:], dh[:, :I], dh[:, I:]
        z = math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)
        gelu = 0.5 * g * (1 + torch.tanh(z))
        a = gelu * u
        d = 1.13 * dg * (u.abs() + du) + gelu.abs() * du + (12 + 8 * z.abs()) * 2.0**-23 * a.abs() + 1e-30
        b, db = blocks_of(a), blocks_of(d)
        s = pow2(scale_exponents(b))
        v, dv = b.abs() / s, db / s
        step = torch.zeros_like(v)
        for m, _ in MIDS:
            step = torch.where((v - m).abs() <= dv, 2.0, step)
        big = v.amax(-1, keepdim=True)
        dbig = torch.where(v + dv >= big, dv, 0.0).amax(-1, keepdim=True)
        step = torch.where(((big - 4).abs() <= dbig) | ((big - 8).abs() <= dbig), 4.0, step)
        da = (step * s).flatten(-2)[..., :I]
        q = mx4_values(a)
        weight = c["probs"][t, k].double() * (c["scale"][e].double() if scaled else 1.0)
        y, ym, yd = q @ dn.t(), q.abs() @ dn.abs().t(), da @ dn.abs().t()
        S = -(-I // 64) + 2
        out.index_add_(0, t, y * weight[:, None])
        mag.index_add_(0, t, ym * weight[:, None])
        tol.index_add_(0, t, (yd + S * 2.0**-23 * (ym + yd)) * weight[:, None])
    # y's own 16-bit or finer storage: at most 2^-15 of a 32-block's largest
    # value, itself below the magnitude sum; then K products and additions
    tol = tol + (K + 3) * 2.0**-24 * mag
    dt = c["x"].dtype
    return out, tol + UNIT[dt] * (out.abs() + tol) + 2.0**-24 * (dt == torch.float16)


LAYERS = [
    # T, K, E, H, I, dropped, all on one expert
    (1, 1, 1, 32, 32, 0.0, None), (1, 8, 128, 256, 96, 0.0, None), (4, 2, 16, 1024, 512, 0.0, None),
    (37, 8, 61, 320, 100, 0.3, None), (64, 8, 128, 256, 704, 0.0, None), (200, 4, 8, 1000, 500, 0.05, None),
    (300, 2, 5, 256, 64, 0.0, 3), (9, 4, 8, 96, 33, 1.0, None), (513, 1, 3, 65, 129, 0.0, None),
    (2048, 2, 16, 256, 128, 0.0, None),
    (700, 4, 8, 416, 352, 0.1, None), (1500, 2, 5, 320, 96, 0.0, 4), (900, 8, 16, 264, 200, 0.2, None),
    (4100, 4, 8, 1088, 700, 0.1, None), (3000, 8, 7, 1040, 333, 0.0, None),
    # few enough pairs for three launches: dropped slots, all dropped, slots that share an expert, the largest
    (1, 8, 128, 2816, 704, 0.0, None), (1, 8, 9, 96, 40, 0.4, None), (2, 4, 8, 320, 100, 1.0, None),
    (3, 4, 16, 1001, 70, 0.0, 5), (4, 8, 32, 2816, 96, 0.1, None), (16, 2, 61, 704, 130, 0.2, None),
    (1, 32, 64, 8192, 64, 0.0, None),
    (16, 8, 128, 1001, 70, 0.2, None), (16, 8, 8, 320, 100, 0.0, 5), (2, 64, 256, 96, 40, 0.3, None),
    (15, 8, 12, 2816, 96, 0.1, None), (9, 14, 60, 96, 65, 0.5, None), (16, 8, 16, 8192, 33, 0.0, None),
    (17, 2, 16, 320, 64, 0.1, None),
    # large batches, more than 8 slots
    (2048, 8, 16, 1024, 64, 0.0, None), (6000, 8, 9, 600, 96, 0.05, None), (1500, 12, 24, 1001, 40, 0.3, None),
    (3200, 8, 16, 1088, 96, 0.1, None), (2500, 12, 24, 1001, 40, 0.3, None),
]


@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("T,K,E,H,I,drop,one", LAYERS)
def test_experts(cuda, moe, T, K, E, H, I, drop, one, dtype):
    c = experts_case(T + H, T, K, E, H, I, dtype, cuda, drop, one)
    out, ws = run_experts(moe, c, T, K, E, H, I)
    assert moe.device_status(ws)[0] == 0
    want, tol = experts_reference(c, T, K, E, H, I)
    assert ((out.double() - want).abs() <= tol).all()
    # again in the used workspace, and with other tokens' contents in between
    other = dict(c, x=c["x"].flip(0), ids=c["ids"].flip(0))
    run_experts(moe, other, T, K, E, H, I, ws=ws)
    again, _ = run_experts(moe, c, T, K, E, H, I, ws=ws)
    assert torch.equal(again, out)
    plain, _ = run_experts(moe, c, T, K, E, H, I, scaled=False)
    want, tol = experts_reference(c, T, K, E, H, I, scaled=False)
    assert ((plain.double() - want).abs() <= tol).all()


def test_experts_strides_graph_and_bad_ids(cuda, moe):
    T, K, E, H, I = 40, 4, 16, 328, 160
    c = experts_case(7, T, K, E, H, I, torch.bfloat16, cuda)
    want, tol = experts_reference(c, T, K, E, H, I)
    _, x = strided(T, H, torch.bfloat16, cuda, 5, 1)
    x.copy_(c["x"])
    buf, out = strided(T, H, torch.bfloat16, cuda, 7, 3, fill=5.0)
    _, ws = run_experts(moe, dict(c, x=x), T, K, E, H, I, out=out)
    assert ((out.double() - want).abs() <= tol).all()
    out.fill_(5.0)
    assert (buf == 5.0).all()
    # a captured call replays on new contents
    s = torch.cuda.Stream()
    qg, qd = quantize(moe, c["gate_up"], gated=True), quantize(moe, c["down"])
    out = torch.zeros(T, H, dtype=torch.bfloat16, device=cuda)
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        moe.mx4_experts(qg, qd, c["ids"], c["probs"], c["scale"], c["x"], out, H, I, E, K, T, ws, stream=s)
    d = experts_case(8, T, K, E, H, I, torch.bfloat16, cuda)
    for n in ("ids", "probs", "x"):
        c[n].copy_(d[n])
    graph.replay()
    torch.cuda.synchronize()
    want, tol = experts_reference(c, T, K, E, H, I)
    assert ((out.double() - want).abs() <= tol).all()
    # an id past the experts is left out and reported, also among a few pairs
    c["ids"][3, 2] = E
    for rows in (T, 4):
        d = dict(c, **{n: c[n][:rows].contiguous() for n in ("ids", "probs", "x")})
        out, ws = run_experts(moe, d, rows, K, E, H, I)
        assert moe.device_status(ws)[0] == -7
        want, tol = experts_reference(d, rows, K, E, H, I)
        assert ((out.double() - want).abs() <= tol).all()


def test_experts_keep_non_finite_tokens_apart(cuda, moe):
    T, K, E, H, I = 33, 2, 4, 128, 64
    c = experts_case(9, T, K, E, H, I, torch.float32, cuda)
    clean, _ = run_experts(moe, c, T, K, E, H, I)
    c["x"] = c["x"].clone()
    c["x"][11, 17] = float("nan")
    c["x"][20, 90] = float("inf")
    out, _ = run_experts(moe, c, T, K, E, H, I)
    bad = torch.zeros(T, dtype=torch.bool, device=cuda)
    bad[[11, 20]] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
