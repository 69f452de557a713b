"""examples/query_decoder.py: the pyramid norm, rotary positions, MSDA and the
8-bit AdamW in one training loop."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "query_decoder.py")


def _example():
    spec = importlib.util.spec_from_file_location("query_decoder", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_decoder_learns():
    losses = _example().train(steps=60)
    assert all(x == x for x in losses)
    # targets of variance 1 that nothing predicts at first
    assert losses[0] > 0.9 and losses[-1] < 0.6 * losses[0]


def test_every_parameter_has_a_gradient():
    ex = _example()
    torch.manual_seed(0)
    shapes = [(8, 8), (4, 4)]
    model = ex.QueryDecoder(shapes, channels=32, queries=10, layers=1).cuda()
    maps = [torch.randn(2, 32, h, w, device="cuda") for h, w in shapes]
    model(maps).square().sum().backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()), name
    assert float(model.places.grad.abs().max()) > 0
