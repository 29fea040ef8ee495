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


@pytest.mark.parametrize("name", ["in_proj", "out_proj"])
def test_a_refused_step_leaves_its_caches(name):
    """A step in place of over 64 rows whose last layer's copy is stale; taken again after its copies are made
    anew it gives what it would have given."""
    torch.manual_seed(6)
    model = Mamba3(128, d_state=32, depth=2).eval().to(DEV, BF16).quantize_prefill()
    x = torch.randn(66, 5, 128, device=DEV, dtype=BF16)
    with torch.no_grad():
        cache = model.prefill(x[:, :4])[1]
        before = [[t.clone() for t in states] for states in cache]
        getattr(model.layers[1].mixer, name).weight.mul_(1)
        with pytest.raises(RuntimeError, match="call it again"):
            model.step(x[:, 4:], cache, inplace=True)
        assert all(torch.equal(a, b) for mine, then in zip(cache, before) for a, b in zip(mine, then))
        model.quantize_prefill()
        got, moved = model.step(x[:, 4:], cache, inplace=True)
        want, other = model.step(x[:, 4:], before)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for mine, then in zip(moved, other) for a, b in zip(mine, then))
