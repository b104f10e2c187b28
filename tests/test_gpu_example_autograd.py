"""The example's autograd functions keep what their own forward pass used."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(cuda):
    spec = importlib.util.spec_from_file_location("mx4_moe_layer", os.path.join(ROOT, "examples", "mx4_moe_layer.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    return ex


def test_two_forward_passes_before_a_backward(cuda, example):
    """Gradients of two passes with other routings, whose backward runs after both, against each pass alone and against
    plain indexing (sums of K = 2 terms in f32: equal but for the order of two additions, which commute)."""
    T, K, E, H = 50, 2, 8, 48
    g = torch.Generator(device=cuda).manual_seed(1)
    ws = example.moe.new_sort_workspace(E, K, T, cuda)
    x = torch.randn(T, H, generator=g, device=cuda)
    ids = [torch.topk(torch.randn(T, E, generator=g, device=cuda), K, 1).indices for _ in range(2)]
    probs = [torch.rand(T, K, generator=g, device=cuda) for _ in range(2)]
    mix = torch.randn(E, H, generator=g, device=cuda)

    def one(i, leaf, p):
        pos, pair = example.sort_tokens(ids[i], E, ws)
        rows = example.Permuted.apply(leaf, pos, pair, H, K, T)
        expert = ids[i].reshape(-1)[pair.long()]
        return example.Unpermuted.apply(rows * mix[expert], p, pos, pair, H, K, T).square().sum()

    def grads(both):
        leaves = [(x.clone().requires_grad_(), p.clone().requires_grad_()) for p in probs]
        if both:
            losses = [one(i, *leaf) for i, leaf in enumerate(leaves)]
            for loss in losses:
                loss.backward()
        else:
            for i, leaf in enumerate(leaves):
                one(i, *leaf).backward()
        return [t.grad for leaf in leaves for t in leaf]

    alone, together = grads(False), grads(True)
    assert all(torch.equal(a, b) for a, b in zip(alone, together))
    for i in range(2):
        leaf, p = x.double().requires_grad_(), probs[i].double().requires_grad_()
        (leaf[:, None] * mix.double()[ids[i]] * p[..., None]).sum(1).square().sum().backward()
        # f32 products and sums of K terms, twice over (the loss' gradient and the way back): within 16 roundings of the
        # magnitudes, which are below the largest entry times a few; H terms in the weights' gradient
        for got, want, n in ((alone[2 * i], leaf.grad, 16), (alone[2 * i + 1], p.grad, 16 + H)):
            assert ((got.double() - want).abs() <= n * 2.0**-24 * 16 * want.abs().max()).all()


def test_changing_what_a_pass_saved_is_noticed(cuda, example):
    T, K, E, H = 6, 2, 4, 8
    ws = example.moe.new_sort_workspace(E, K, T, cuda)
    x = torch.randn(T, H, device=cuda, requires_grad=True)
    pos, pair = example.sort_tokens(torch.topk(torch.randn(T, E, device=cuda), K, 1).indices, E, ws)
    rows = example.Permuted.apply(x, pos, pair, H, K, T)
    pos.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        rows.sum().backward()
