"""``Mamba3.quantize_prefill``: what a model that is held in 8 bits refuses, and what it leaves as it was."""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import Mamba3

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16 = torch.bfloat16


def test_graphs_from_before_are_refused():
    torch.manual_seed(5)
    model = Mamba3(128, d_state=32, depth=2).eval().to(DEV, BF16)
    x = torch.randn(70, 1, 128, device=DEV, dtype=BF16)
    few, many = model.cuda_graph(3), model.cuda_graph(70)
    want = few(x[:3], validate=True).clone()
    many(x, validate=True)
    model.quantize_prefill()
    few.reset()
    assert torch.equal(few(x[:3], validate=True), want)
    with pytest.raises(RuntimeError, match="recreate"):
        many(x, validate=True)
    fresh = model.cuda_graph(70)
    got = fresh(x, validate=True).clone()
    model.quantize_prefill()
    fresh.reset()
    assert torch.equal(fresh(x, validate=True), got)
    with torch.inference_mode():
        assert torch.equal(model.step(x)[0], got)
