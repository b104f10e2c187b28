"""The example runs: MXFP4 serving stays near the exact layer, and a training
loop through the permutation and MXFP4 operators lowers its loss."""

from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_example(cuda):
    spec = importlib.util.spec_from_file_location("mx4_moe_layer", os.path.join(ROOT, "examples", "mx4_moe_layer.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    # E2M1 rounds to within a quarter of a value's binade, about 0.1 of it in the mean square; three quantised
    # factors per product and as many again for Q4_0's own values keep the layer's difference below 0.5
    assert all(0.0 < d < 0.5 for d in ex.serve(cuda, batches=(1, 64, 300)).values())
    losses = ex.train(cuda)
    assert losses[-1] < 0.8 * losses[0]
