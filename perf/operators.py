"""Workloads of the token-permutation and MXFP4 operators, for timing and for checking their outputs.

Five operators, each as a user's program calls it:

  permute    the (token, slot) pairs sorted by expert, and the tokens' rows gathered in that order; with
             "train" also the gradient of the tokens from the gradient of the gathered rows
  unpermute  the experts' rows back in token order, weighted and summed over the slots; with "train" also the
             gradients of the rows and of the weights
  quantize   a matrix to MXFP4 (blocks of 32 E2M1 values with one power-of-two scale) and the values it stands
             for; with "both" also its transpose, quantised along the other axis
  linear     a linear layer in MXFP4: the input quantised, then the product with quantised weights; with "train"
             also the input's and the weights' gradients, every operand quantised along its summed axis
  experts    a mixture-of-experts FFN layer in MXFP4 after routing: sort, quantise, gate/up products with GeGLU,
             down products, weighted sum

`own` chooses between the plain form (elementary torch operations in 32 bits) and the library's kernels.
"""

from __future__ import annotations

import math
import os

import torch

own = False

HERE = os.path.dirname(os.path.abspath(__file__))
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32  # values that share a scale
MX_BYTES = 17 / 32  # bytes of an MXFP4 value, its share of the scale included

_lib = None


def library():
    """The package's operator module (its folder's name is no identifier)."""
    global _lib
    if _lib is None:
        import importlib.util
        import sys

        path = os.path.join(os.path.dirname(HERE), "qt_llama.cpp_b200", "mrml_moe.py")
        spec = importlib.util.spec_from_file_location("mrml_moe_b200", path)
        _lib = importlib.util.module_from_spec(spec)
        sys.modules["mrml_moe_b200"] = _lib
        spec.loader.exec_module(_lib)
    return _lib


# ---------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # A decode step's eight tokens of the 128-expert layer, sorted and gathered for experts of one's own.
        dict(name="permute_decode", op="permute", T=8, K=8, E=128, H=2816, dtype="bf16", drop=0.0, train=False),
        # A training batch of the same layer: gather, and the gradient back to the tokens.
        dict(name="permute_train", op="permute", T=8192, K=8, E=128, H=2816, dtype="bf16", drop=0.0, train=True),
        # The 16-expert layer's shape made odd, in 32 bits, with slots that a capacity limit dropped.
        dict(name="permute_odd", op="permute", T=1531, K=2, E=16, H=1001, dtype="f32", drop=0.1, train=True),
        # The weighted sum of a decode batch of 64.
        dict(name="unpermute_decode", op="unpermute", T=64, K=8, E=128, H=2816, dtype="f32", drop=0.0, train=False),
        # The same for a training batch, with the gradients of the experts' rows and of the routing weights.
        dict(name="unpermute_train", op="unpermute", T=8192, K=8, E=128, H=2816, dtype="bf16", drop=0.02, train=True),
        # A few rows of a ragged width, as activations come in at decode.
        dict(name="quantize_ragged", op="quantize", rows=33, cols=1000, dtype="f16", both=False),
        # Sixteen experts' gate and up weights, quantised for both directions of a training step.
        dict(name="quantize_weights", op="quantize", rows=22528, cols=2816, dtype="bf16", both=True),
        # One token through the shared MLP's gate and up rows.
        dict(name="linear_token", op="linear", T=1, N=4224, K=2816, dtype="bf16", train=False),
        # A training step of the same linear layer on 4096 tokens: forward and both gradients.
        dict(name="linear_train", op="linear", T=4096, N=4224, K=2816, dtype="bf16", train=True),
        # The whole 128-expert layer: one token, a decode batch, a long prompt.
        dict(name="experts_token", op="experts", T=1, K=8, E=128, H=2816, I=704, dtype="bf16"),
        dict(name="experts_decode", op="experts", T=64, K=8, E=128, H=2816, I=704, dtype="bf16"),
        dict(name="experts_prompt", op="experts", T=8192, K=8, E=128, H=2816, I=704, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["permute", "unpermute", "quantize", "linear", "experts"])
    if op in ("permute", "unpermute"):
        E = rng.choice([8, 16, 61, 128])
        H = rng.choice([256, 1000, 1024, 1537, 2816])
        return dict(op=op, T=_spread(rng, 1, 8192), K=rng.choice([1, 2, 4, 6, 8]), E=E, H=H,
                    dtype=rng.choice(["f16", "bf16"]) if H > 1100 else rng.choice(["f32", "f16", "bf16"]),
                    drop=rng.choice([0.0, 0.0, 0.05, 0.3]), train=rng.random() < 0.5)
    if op == "quantize":
        return dict(op=op, rows=_spread(rng, 1, 16384), cols=_spread(rng, 20, 2816),
                    dtype=rng.choice(["f32", "f16", "bf16"]), both=rng.random() < 0.5)
    if op == "linear":
        return dict(op=op, T=_spread(rng, 1, 4096), N=_spread(rng, 60, 4224), K=_spread(rng, 60, 2816),
                    dtype=rng.choice(["f16", "bf16"]), train=rng.random() < 0.4)
    return dict(op=op, T=_spread(rng, 1, 4096), K=rng.choice([1, 2, 4, 8]), E=rng.choice([8, 16, 60, 128]),
                H=rng.choice([256, 1000, 1024, 2048, 2816]), I=rng.choice([96, 500, 512, 704]),
                dtype=rng.choice(["f16", "bf16"]))


def work(case):
    c, s = case, SIZE[case["dtype"]]
    if c["op"] in ("permute", "unpermute"):
        pairs, x, rows = c["T"] * c["K"], c["T"] * c["H"] * s, c["T"] * c["K"] * c["H"] * s
        if c["op"] == "permute":  # ids in, places and rows out; then the rows' gradient in, the tokens' out
            n = 12 * pairs + x + rows + (rows + x if c["train"] else 0)
            return {"bytes": n, "flops": pairs * c["H"] if c["train"] else 0}
        # rows and weights in, tokens out; then the tokens' gradient in, the rows' and the weights' out
        n = 8 * pairs + rows + x + (x + rows + 4 * pairs if c["train"] else 0)
        return {"bytes": n, "flops": (5 if c["train"] else 2) * pairs * c["H"]}
    if c["op"] == "quantize":
        n, value = c["rows"] * c["cols"], 4 if c["dtype"] == "f32" else 2
        return {"bytes": n * s + (2 if c["both"] else 1) * n * (value + MX_BYTES), "flops": 4 * n}
    if c["op"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        if c["train"]:
            return {"bytes": 2 * s * (T * K + T * N + N * K), "flops": 6 * T * N * K}
        return {"bytes": s * (T * K + T * N) + N * K * MX_BYTES, "flops": 2 * T * N * K}
    T, K, E, H, I = c["T"], c["K"], c["E"], c["H"], c["I"]
    hit = E * (1 - (1 - K / E) ** T)  # experts that a batch is expected to reach
    return {"bytes": hit * 3 * H * I * MX_BYTES + 2 * T * H * s + 8 * T * K, "flops": 6 * T * K * H * I}


# --------------------------------------------------------------------------------------------------- inputs


def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def _tokens(g, T, H):
    """Hidden states: normal, with a few channels that run larger, as they do in trained models."""
    gain = torch.exp(0.3 * _normal(g, H))
    gain[torch.rand(H, generator=g, device="cuda") < 0.01] *= 8.0
    return _normal(g, T, H) * gain


def _routing(g, T, K, E, drop):
    """ids [T][K] (distinct per token, -1 where dropped) and their renormalised weights, skewed over the experts."""
    bias = -0.5 * torch.log(1.0 + torch.randperm(E, generator=g, device="cuda").float())
    top, ids = torch.topk(_normal(g, T, E) + bias, K, dim=1)
    probs = torch.softmax(top, dim=1)
    ids = ids.to(torch.int32)
    if drop:
        ids = torch.where(torch.rand(T, K, generator=g, device="cuda") < drop, torch.full_like(ids, -1), ids)
    return ids, probs


def _inputs(case, seed):
    """The case's data, the same for every form."""
    c, g, dt = case, _generator(case, seed), DTYPES[case["dtype"]]
    d = {}
    if c["op"] in ("permute", "unpermute"):
        d["ids"], d["probs"] = _routing(g, c["T"], c["K"], c["E"], c["drop"])
        if c["op"] == "permute":
            d["x"] = _tokens(g, c["T"], c["H"]).to(dt)
        d["rows"] = _normal(g, c["T"] * c["K"], c["H"]).to(dt)  # the experts' rows, or the gathered rows' gradient
        if c["op"] == "unpermute" and c["train"]:
            d["dout"] = _normal(g, c["T"], c["H"]).to(dt)
    elif c["op"] == "quantize":
        d["x"] = _tokens(g, c["rows"], c["cols"]).to(dt)
    elif c["op"] == "linear":
        d["x"] = _tokens(g, c["T"], c["K"]).to(dt)
        d["w"] = _normal(g, c["N"], c["K"], std=0.02).to(dt)
        if c["train"]:
            d["dy"] = _normal(g, c["T"], c["N"]).to(dt)
    else:
        d["ids"], d["probs"] = _routing(g, c["T"], c["K"], c["E"], 0.0)
        d["scale"] = torch.rand(c["E"], generator=g, device="cuda") + 0.5
        d["x"] = _tokens(g, c["T"], c["H"]).to(dt)
        d["gate_up"] = _normal(g, c["E"], 2 * c["I"], c["H"], std=0.02).to(dt)
        d["down"] = _normal(g, c["E"], c["H"], c["I"], std=0.05).to(dt)
    return d


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    s = dict(case=dict(case), **d)
    if c["op"] == "unpermute":  # the sort of the forward pass, kept for the way back
        s.update(_sort(d["ids"], c["E"]))
    # Weights are quantised once, when a model is loaded; a training step quantises them anew each time.
    if c["op"] == "linear" and not c["train"]:
        s["w"] = _keep(s["w"][None], False)
    if c["op"] == "experts":
        s["gate_up"], s["down"] = _keep(s["gate_up"], True), _keep(s["down"], False)
    if own:
        m, dev = library(), torch.device("cuda")
        if c["op"] == "permute":
            s["ws"] = m.new_sort_workspace(c["E"], c["K"], c["T"], dev)
        if c["op"] == "linear":
            T, N, K = c["T"], c["N"], c["K"]
            s["ws"] = m.new_mx4_linear_workspace(T, N, K, dev)
            if c["train"]:
                s["q"] = {n: m.new_mx4(r, k, 1, dev) for n, r, k in (
                    ("x", T, K), ("xt", K, T), ("w", N, K), ("wt", K, N), ("dy", T, N), ("dyt", N, T))}
        if c["op"] == "experts":
            s["ws"] = m.new_mx4_experts_workspace(c["H"], c["I"], c["E"], c["K"], c["T"], dev)
        if c["op"] == "quantize":
            s["q"] = m.new_mx4(c["rows"], c["cols"], 1, dev)
            s["qt"] = m.new_mx4(c["cols"], c["rows"], 1, dev) if c["both"] else None
    return s


def _keep(w, gated):
    """Quantised weights as each form keeps them: the library's buffer, or the values in 32 bits."""
    if not own:
        return _mx4(w)
    m = library()
    n, rows, cols = w.shape
    q = m.new_mx4(rows, cols, n, w.device)
    m.mx4_quantize(w, q, rows, cols, n, gated=gated)
    return q


# ----------------------------------------------------------------------------------------------- plain form


def _mx4(x):
    """The values of x (32 bits) after MXFP4 quantisation along its last axis.  A block's scale is
    2^(floor(log2(max |x|)) - 2), at least 2^-127; values round to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times
    it (ties to the even one), at most 6."""
    x = x.float()
    cols = x.shape[-1]
    pad = -cols % BLOCK
    if pad:
        x = torch.nn.functional.pad(x, (0, pad))
    b = x.unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(dim=-1, keepdim=True)
    scale = torch.exp2((torch.frexp(amax).exponent - 3).clamp(min=-127).float() + 32) * 2.0**-32
    v = b / scale
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.round(v / step) * step
    return (q.clamp(-6, 6) * scale).flatten(-2)[..., :cols]


def _sort(ids, E):
    """Pairs in expert order: where each expert starts, how many it has, each pair's place (-1: none) and each
    place's pair (-1: none)."""
    T, K = ids.shape
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(E, device=ids.device)).sum(0)
    ends = counts.cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(T * K, device=ids.device)
    total = ends[-1]
    pos = torch.where(key < E, place, -1)
    pair = torch.where(torch.arange(T * K, device=ids.device) < total, order, -1)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    return {n: v.to(torch.int32) for n, v in
            dict(offsets=offsets, counts=counts, pos=pos.reshape(T, K), pair=pair).items()}


def _rows_of(rows, pos):
    """[T][K][H] in 32 bits: each pair's row, zero where it has none."""
    got = rows[pos.clamp(min=0).long()].float()
    return torch.where(pos[..., None] >= 0, got, 0.0)


def _plain_permute(s):
    c, x = s["case"], s["x"]
    out = _sort(s["ids"], c["E"])
    pair = out["pair"].long()
    out["out"] = torch.where(pair[:, None] >= 0, x[pair.clamp(min=0) // c["K"]], torch.zeros_like(x[:1]))
    if c["train"]:
        out["dx"] = _rows_of(s["rows"], out["pos"]).sum(1).to(x.dtype)
    return out


def _plain_unpermute(s):
    c, rows, pos, probs = s["case"], s["rows"], s["pos"], s["probs"]
    y = _rows_of(rows, pos)
    out = {"out": (y * probs[..., None]).sum(1).to(rows.dtype)}
    if c["train"]:
        dout = s["dout"].float()
        out["dprobs"] = (y * dout[:, None, :]).sum(-1)
        pair = s["pair"].long().clamp(min=0)
        d = dout[pair // c["K"]] * probs.reshape(-1)[pair][:, None]
        out["drows"] = torch.where(s["pair"][:, None] >= 0, d, 0.0).to(rows.dtype)
    return out


def _plain_quantize(s):
    x = s["x"]
    dt = torch.float32 if x.dtype == torch.float32 else torch.bfloat16
    out = {"values": _mx4(x).to(dt)}
    if s["case"]["both"]:
        out["values_t"] = _mx4(x.t()).to(dt)
    return out


def _plain_linear(s):
    c, x = s["case"], s["x"]
    if not c["train"]:
        return {"y": (_mx4(x) @ s["w"][0].t()).to(x.dtype)}
    w, dy = s["w"], s["dy"]
    return {"y": (_mx4(x) @ _mx4(w).t()).to(x.dtype),
            "dx": (_mx4(dy) @ _mx4(w.t()).t()).to(x.dtype),
            "dw": (_mx4(dy.t()) @ _mx4(x.t()).t()).to(x.dtype)}


def _gelu(v):
    return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _plain_experts(s):
    c, x = s["case"], s["x"]
    E, K, I = c["E"], c["K"], c["I"]
    o = _sort(s["ids"], E)
    room = int(o["counts"].max())
    ids = s["ids"].long().reshape(-1)
    slot = o["pos"].reshape(-1).long() - o["offsets"].long()[ids]  # a pair's place among its expert's
    token = torch.arange(c["T"] * K, device=x.device) // K
    batch = torch.zeros(E, room, c["H"], device=x.device)
    batch[ids, slot] = _mx4(x)[token]
    h = torch.bmm(batch, s["gate_up"].transpose(1, 2))
    act = _mx4(_gelu(h[..., :I]) * h[..., I:])
    y = torch.bmm(act, s["down"].transpose(1, 2))[ids, slot].reshape(c["T"], K, c["H"])
    weight = s["probs"] * s["scale"][s["ids"].long()]
    return {"out": (y * weight[..., None]).sum(1).to(x.dtype)}


_PLAIN = {"permute": _plain_permute, "unpermute": _plain_unpermute, "quantize": _plain_quantize,
          "linear": _plain_linear, "experts": _plain_experts}


# ------------------------------------------------------------------------------------------ the library's form


def _own_permute(s):
    m, c, x = library(), s["case"], s["x"]
    T, K, E, H = c["T"], c["K"], c["E"], c["H"]
    n = m.sorted_rows(E, K, T)
    i32 = dict(dtype=torch.int32, device=x.device)
    out = dict(offsets=torch.empty(E + 1, **i32), counts=torch.empty(E, **i32), pos=torch.empty(T, K, **i32),
               pair=torch.empty(n, **i32), out=torch.empty(n, H, dtype=x.dtype, device=x.device))
    m.sort(s["ids"], out["offsets"], out["counts"], out["pos"], out["pair"], E, K, T, 1, s["ws"])
    m.permute(x, out["pair"], out["out"], H, K)
    if c["train"]:
        out["dx"] = torch.empty_like(x)
        m.permute_grad(s["rows"], out["pos"], out["dx"], H, K, T)
    return out


def _own_unpermute(s):
    m, c, rows = library(), s["case"], s["rows"]
    T, K, H = c["T"], c["K"], c["H"]
    out = {"out": torch.empty(T, H, dtype=rows.dtype, device=rows.device)}
    m.unpermute(rows, s["pos"], s["probs"], out["out"], H, K, T)
    if c["train"]:
        out["drows"], out["dprobs"] = torch.empty_like(rows), torch.empty_like(s["probs"])
        m.unpermute_grad(s["dout"], rows, s["pos"], s["pair"], s["probs"], out["drows"], out["dprobs"], H, K, T)
    return out


def _own_quantize(s):
    m, c, x = library(), s["case"], s["x"]
    r, k = c["rows"], c["cols"]
    dt = torch.float32 if x.dtype == torch.float32 else torch.bfloat16
    out = {"values": torch.empty(r, k, dtype=dt, device=x.device)}
    if c["both"]:
        out["values_t"] = torch.empty(k, r, dtype=dt, device=x.device)
        m.mx4_quantize_both(x, s["q"], s["qt"], r, k)
        m.mx4_dequantize(s["qt"], out["values_t"], k, r)
    else:
        m.mx4_quantize(x, s["q"], r, k)
    m.mx4_dequantize(s["q"], out["values"], r, k)
    return out


def _own_linear(s):
    m, c, x = library(), s["case"], s["x"]
    T, N, K = c["T"], c["N"], c["K"]
    y = torch.empty(T, N, dtype=x.dtype, device=x.device)
    if not c["train"]:
        m.mx4_linear(x, s["w"], y, T, N, K, s["ws"])
        return {"y": y}
    q, dx, dw = s["q"], torch.empty_like(x), torch.empty_like(s["w"])
    m.mx4_quantize_both(x, q["x"], q["xt"], T, K)
    m.mx4_quantize_both(s["w"], q["w"], q["wt"], N, K)
    m.mx4_matmul(q["x"], q["w"], y, T, N, K, s["ws"])
    m.mx4_quantize_both(s["dy"], q["dy"], q["dyt"], T, N)
    m.mx4_matmul(q["dy"], q["wt"], dx, T, K, N, s["ws"])
    m.mx4_matmul(q["dyt"], q["xt"], dw, N, K, T, s["ws"])
    return {"y": y, "dx": dx, "dw": dw}


def _own_experts(s):
    m, c, x = library(), s["case"], s["x"]
    out = torch.empty_like(x)
    m.mx4_experts(s["gate_up"], s["down"], s["ids"], s["probs"], s["scale"], x, out, c["H"], c["I"], c["E"], c["K"],
                  c["T"], s["ws"])
    return {"out": out}


_OWN = {"permute": _own_permute, "unpermute": _own_unpermute, "quantize": _own_quantize, "linear": _own_linear,
        "experts": _own_experts}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------- 64 bits


def _exact_mx4(x):
    """MXFP4 values in 64 bits, from the format's table and its midpoints."""
    x = x.double()
    cols = x.shape[-1]
    out = torch.zeros(*x.shape[:-1], -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    out[..., :cols] = x
    b = out.reshape(*x.shape[:-1], -1, BLOCK)
    big = b.abs().max(dim=-1, keepdim=True).values
    e = ((big.view(torch.int64) >> 52) - 1023 - 2).clamp(min=-127)  # a double's own exponent
    scale = ((e + 1023) << 52).view(torch.float64)
    a = b.abs() / scale
    code = ((a > 0.25).long() + (a >= 0.75).long() + (a > 1.25).long() + (a >= 1.75).long() + (a > 2.5).long()
            + (a >= 3.5).long() + (a > 5.0).long())
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    return (torch.sign(b) * table[code] * scale).reshape(out.shape)[..., :cols]


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    op = c["op"]
    if op == "quantize":
        out = {"values": _exact_mx4(d["x"])}
        if c["both"]:
            out["values_t"] = _exact_mx4(d["x"].t())
        return out
    if op == "linear":
        x, w = _exact_mx4(d["x"]), _exact_mx4(d["w"])
        out = {"y": x @ w.t()}
        if c["train"]:
            out["dx"] = _exact_mx4(d["dy"]) @ _exact_mx4(d["w"].t()).t()
            out["dw"] = _exact_mx4(d["dy"].t()) @ _exact_mx4(d["x"].t()).t()
        return out
    ids, T, K = d["ids"].long(), c["T"], c["K"]
    if op == "experts":
        x = _exact_mx4(d["x"])
        out = torch.zeros(T, c["H"], dtype=torch.float64, device=x.device)
        for e in range(c["E"]):
            token, slot = torch.nonzero(ids == e, as_tuple=True)
            if not len(token):
                continue
            h = x[token] @ _exact_mx4(d["gate_up"][e]).t()
            g, u = h[:, :c["I"]], h[:, c["I"]:]
            act = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
            y = _exact_mx4(act) @ _exact_mx4(d["down"][e]).t()
            out.index_add_(0, token, y * (d["probs"][token, slot].double() * d["scale"][e].double())[:, None])
        return {"out": out}
    # Places by counting: pairs of earlier experts, then earlier pairs of the same one.
    flat = ids.reshape(-1)
    starts, place, at = [0], torch.full_like(flat, -1), 0
    for e in range(c["E"]):
        mine = torch.nonzero(flat == e).reshape(-1)
        place[mine] = at + torch.arange(len(mine), device=flat.device)
        at += len(mine)
        starts.append(at)
    pos = place.reshape(T, K)
    if op == "permute":
        n = T * K
        pair = torch.full((n,), -1, dtype=torch.long, device=flat.device)
        kept = torch.nonzero(place >= 0).reshape(-1)
        pair[place[kept]] = kept
        rows = torch.zeros(n, c["H"], dtype=torch.float64, device=flat.device)
        rows[place[kept]] = d["x"].double()[kept // K]
        ends = torch.tensor(starts, dtype=torch.int32, device=flat.device)
        out = {"offsets": ends, "counts": ends[1:] - ends[:-1], "pos": pos.int(), "pair": pair.int(), "out": rows}
        if c["train"]:
            out["dx"] = torch.zeros(T, c["H"], dtype=torch.float64, device=flat.device)
            for k in range(K):
                has = pos[:, k] >= 0
                out["dx"][has] += d["rows"].double()[pos[has, k]]
        return out
    total = torch.zeros(T, c["H"], dtype=torch.float64, device=flat.device)
    drows = torch.zeros(T * K, c["H"], dtype=torch.float64, device=flat.device)
    dprobs = torch.zeros(T, K, dtype=torch.float64, device=flat.device)
    for k in range(K):
        has = pos[:, k] >= 0
        y, p = d["rows"].double()[pos[has, k]], d["probs"][has, k].double()
        total[has] += p[:, None] * y
        if c["train"]:
            g = d["dout"].double()[has]
            drows[pos[has, k]] = p[:, None] * g
            dprobs[has, k] = (y * g).sum(1)
    return {"out": total, "drows": drows, "dprobs": dprobs} if c["train"] else {"out": total}
