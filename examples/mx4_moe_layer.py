"""A mixture-of-experts layer with the permutation and MXFP4 operators.

Serving: the exact router picks the experts, and mx4_experts runs the layer on
MXFP4 weights (quantised here from a GGUF-style Q4_0 slab, as a loaded model
has it), one token, a decode batch, a prompt; each step is one CUDA graph.

Training: experts of one's own between the gather and the weighted sum, with
the library's gradients on the way back: the tokens are sorted by expert,
gathered, sent through one MXFP4 linear layer per direction (forward, and the
gradients of its input and weights), brought back with the routing weights,
and plain gradient steps lower the loss.

    python examples/mx4_moe_layer.py
"""

from __future__ import annotations

import importlib.util
import os

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load(name, *path):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, *path))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


moe = load("mrml_moe_b200", "qt_llama.cpp_b200", "mrml_moe.py")
synth = load("mrml_moe_b200_synth", "qt_llama.cpp_b200", "synth.py")


class Mx4MoeLayer:
    """Router and experts of one layer for up to T tokens; its weights are
    quantised once, from GGUF expert slabs as load_moe_layer returns them."""

    def __init__(self, router_w, gate_up, down, wtype, H, I, E, K, T, device):
        self.shape, self.router_w = (H, I, E, K, T), router_w
        self.gate_up = moe.new_mx4(2 * I, H, E, device)
        self.down = moe.new_mx4(H, I, E, device)
        moe.mx4_quantize(gate_up, self.gate_up, 2 * I, H, E, gated=True, wtype=wtype)
        moe.mx4_quantize(down, self.down, H, I, E, wtype=wtype)
        self.x = torch.zeros(T, H, device=device)
        self.out = torch.zeros(T, H, device=device)
        self.logits = torch.empty(T, E, device=device)
        self.ids = torch.empty(T, K, dtype=torch.int32, device=device)
        self.probs = torch.empty(T, K, device=device)
        self.router_ws = moe.new_workspace(32, 32, E, K, T, device)
        self.ws = moe.new_mx4_experts_workspace(H, I, E, K, T, device)
        stream = torch.cuda.Stream(device)
        stream.wait_stream(torch.cuda.current_stream(device))
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=stream):
            moe.router(self.router_w, self.x, self.logits, self.ids, self.probs, H, E, K, T, self.router_ws, stream)
            moe.mx4_experts(self.gate_up, self.down, self.ids, self.probs, None, self.x, self.out, H, I, E, K, T,
                            self.ws, stream)

    def step(self, x):
        self.x.copy_(x)
        self.graph.replay()
        return self.out


def serve(device, H=1024, I=512, E=16, K=2, batches=(1, 64, 2048)):
    gate_up, down = synth.expert_weights(1, moe.MRML_Q4_0, H, I, E)
    gate_up, down = torch.from_numpy(gate_up).to(device), torch.from_numpy(down).to(device)
    router_w = torch.from_numpy(synth.normal(2, E * H, 0.02).reshape(E, H)).to(device)
    outs = {}
    for T in batches:
        layer = Mx4MoeLayer(router_w, gate_up, down, moe.MRML_Q4_0, H, I, E, K, T, device)
        x = torch.from_numpy(synth.normal(3, T * H).reshape(T, H)).to(device)
        # the same layer in the exact GGUF arithmetic, to see what four bits cost
        exact = torch.empty(T, H, device=device)
        ws = moe.new_workspace(H, I, E, K, T, device)
        out = layer.step(x)
        moe.experts(moe.MRML_Q4_0, gate_up, down, layer.ids, layer.probs, None, x, exact, H, I, E, K, T, ws)
        outs[T] = ((out - exact).norm() / exact.norm()).item()
        print(f"serving {T:5d} tokens: rel. difference to the exact Q4_0 layer {outs[T]:.3f}")
    return outs


def sort_tokens(ids, E, ws):
    """pos and pair of the tokens' experts, in tensors of their own: gradients need those of their own pass, and
    autograd does not see the library write into a buffer that is used again."""
    T, K = ids.shape
    i32 = dict(dtype=torch.int32, device=ids.device)
    offsets, counts = torch.empty(E + 1, **i32), torch.empty(E, **i32)
    pos, pair = torch.empty(T, K, **i32), torch.empty(moe.sorted_rows(E, K, T), **i32)
    moe.sort(ids.to(torch.int32).contiguous(), offsets, counts, pos, pair, E, K, T, 1, ws)
    return pos, pair


class Permuted(torch.autograd.Function):
    """Tokens gathered in expert order, and the gradient back to them."""

    @staticmethod
    def forward(ctx, x, pos, pair, H, K, T):
        ctx.save_for_backward(pos)
        ctx.shape = (H, K, T)
        rows = torch.empty(pair.numel(), H, dtype=x.dtype, device=x.device)
        moe.permute(x, pair, rows, H, K)
        return rows

    @staticmethod
    def backward(ctx, drows):
        (pos,), (H, K, T) = ctx.saved_tensors, ctx.shape
        dx = torch.empty(T, H, dtype=drows.dtype, device=drows.device)
        moe.permute_grad(drows.contiguous(), pos, dx, H, K, T)
        return dx, None, None, None, None, None


class Unpermuted(torch.autograd.Function):
    """Rows weighted and summed per token, and both gradients."""

    @staticmethod
    def forward(ctx, rows, probs, pos, pair, H, K, T):
        ctx.save_for_backward(rows, probs, pos, pair)
        ctx.shape = (H, K, T)
        out = torch.empty(T, H, dtype=rows.dtype, device=rows.device)
        moe.unpermute(rows, pos, probs, out, H, K, T)
        return out

    @staticmethod
    def backward(ctx, dout):
        (rows, probs, pos, pair), (H, K, T) = ctx.saved_tensors, ctx.shape
        drows, dprobs = torch.empty_like(rows), torch.empty_like(probs)
        moe.unpermute_grad(dout.contiguous(), rows, pos, pair, probs, drows, dprobs, H, K, T)
        return drows, dprobs, None, None, None, None, None


class Mx4Linear(torch.autograd.Function):
    """y = x w^T with every operand quantised along its summed axis, in all
    three products (the quantisation itself passes gradients straight on)."""

    @staticmethod
    def forward(ctx, x, w):
        (T, K), N = x.shape, w.shape[0]
        q = [moe.new_mx4(r, c, 1, x.device) for r, c in ((T, K), (K, T), (N, K), (K, N))]
        moe.mx4_quantize_both(x, q[0], q[1], T, K)
        moe.mx4_quantize_both(w, q[2], q[3], N, K)
        y = torch.empty(T, N, dtype=x.dtype, device=x.device)
        moe.mx4_matmul(q[0], q[2], y, T, N, K, moe.new_mx4_matmul_workspace(T, N, K, x.device))
        ctx.save_for_backward(q[1], q[3])
        ctx.shape = (T, N, K)
        return y

    @staticmethod
    def backward(ctx, dy):
        (T, N, K), (xt, wt), dev = ctx.shape, ctx.saved_tensors, dy.device
        dy = dy.contiguous()
        d, dt = moe.new_mx4(T, N, 1, dev), moe.new_mx4(N, T, 1, dev)
        moe.mx4_quantize_both(dy, d, dt, T, N)
        dx = torch.empty(T, K, dtype=dy.dtype, device=dev)
        dw = torch.empty(N, K, dtype=dy.dtype, device=dev)
        moe.mx4_matmul(d, wt, dx, T, K, N, moe.new_mx4_matmul_workspace(T, K, N, dev))
        moe.mx4_matmul(dt, xt, dw, N, K, T, moe.new_mx4_matmul_workspace(N, K, T, dev))
        return dx, dw


def train(device, T=512, H=256, E=8, K=2, steps=12, lr=0.15):
    """A shared map between gather and weighted sum, and a router, learn to
    reproduce the tokens; returns the losses."""
    g = torch.Generator(device=device).manual_seed(0)
    x = torch.randn(T, H, generator=g, device=device)
    w = (0.02 * torch.randn(H, H, generator=g, device=device)).requires_grad_()
    router = (0.1 * torch.randn(E, H, generator=g, device=device)).requires_grad_()
    ws = moe.new_sort_workspace(E, K, T, device)
    losses = []
    for _ in range(steps):
        top, ids = torch.topk(x @ router.t(), K, dim=1)
        pos, pair = sort_tokens(ids, E, ws)
        rows = Mx4Linear.apply(Permuted.apply(x, pos, pair, H, K, T), w)
        out = Unpermuted.apply(rows, torch.softmax(top, 1), pos, pair, H, K, T)
        loss = (out - x).square().mean()
        loss.backward()
        with torch.no_grad():
            for p in (w, router):
                p -= lr * p.grad * (H if p is w else 1.0)
                p.grad = None
        losses.append(loss.item())
    print("training losses:", " ".join(f"{v:.3f}" for v in losses))
    return losses


if __name__ == "__main__":
    serve(torch.device("cuda", 0))
    train(torch.device("cuda", 0))
