"""``in_proj`` and ``out_proj`` that are more than their weight's product (a hook, a bias, a module around them):
what stands in for them elsewhere, a kernel on the weight or a copy of it in fewer bits, passes none of that by."""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import Mamba3, ops

BF16 = torch.bfloat16


class _Adapter(torch.nn.Module):
    """A projection with something beside it, under the projection's own weight."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    @property
    def weight(self):
        return self.inner.weight

    def forward(self, x):
        return self.inner(x) + 1


def _adapted(mixer, name):
    setattr(mixer, name, _Adapter(getattr(mixer, name)))


def _biased(mixer, name):
    weight = getattr(mixer, name).weight
    setattr(mixer, name, torch.nn.Linear(weight.shape[1], weight.shape[0]))


def _hooked(mixer, name):
    getattr(mixer, name).register_forward_hook(lambda module, args, out: out + 1)


def _hooked_before(mixer, name):
    getattr(mixer, name).register_forward_pre_hook(lambda module, args: (args[0] + 1,))


def _patched(mixer, name):
    module = getattr(mixer, name)
    module.forward = lambda x: torch.nn.Linear.forward(module, x) + 1


CHANGES = [_adapted, _biased, _hooked, _hooked_before, _patched]


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("name", ["in_proj", "out_proj"])
def test_quantize_prefill_passes_nothing_by(name, change):
    """A projection that is more than its weight's product is not replaced by its copy: neither one that is so
    when the copies are made, nor one that becomes so afterwards."""
    model = Mamba3(64, depth=2)
    change(model.layers[1].mixer, name)
    with pytest.raises(ValueError, match=f"{name} to be a plain nn.Linear"):
        model.quantize_prefill()
    assert not any(layer.mixer._prefill8 for layer in model.layers)
    model = Mamba3(64, depth=2).quantize_prefill()
    change(model.layers[0].mixer, name)
    with pytest.raises(RuntimeError, match=f"{name}.* changed since quantize_prefill"):
        model.layers[0].mixer._weight8(name)
    if name == "in_proj":
        with pytest.raises(RuntimeError, match="changed since quantize_prefill"), torch.no_grad():
            model(torch.zeros(1, 2, 64))


def test_quantize_prefill_takes_linears_of_another_name():
    class Own(torch.nn.Linear):
        pass

    model = Mamba3(64, depth=1)
    mixer = model.layers[0].mixer
    mixer.out_proj = Own(128, 64, bias=False)
    assert model.quantize_prefill() is model and mixer._weight8("out_proj") is not None


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("name", ["in_proj", "out_proj"])
def test_quantize_decode_passes_nothing_by(name, change):
    model = Mamba3(64, depth=2).to(BF16)
    change(model.layers[1].mixer, name)
    model.to(BF16)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    with pytest.raises(ValueError, match=f"{name} to be a plain nn.Linear"):
        model.quantize_decode(32)
    assert not any(layer.mixer._decode4 for layer in model.layers)
    assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items())
    model = Mamba3(64, depth=2).to(BF16).quantize_decode(32)
    change(model.layers[0].mixer, name)
    with pytest.raises(RuntimeError, match=f"{name}.* changed since quantize_decode"):
        model.layers[0].mixer._weight4(name)


@pytest.mark.parametrize("change", [None, *CHANGES])
@pytest.mark.parametrize("name", ["in_proj", "out_proj"])
def test_a_step_passes_nothing_by(monkeypatch, name, change):
    """With a decode kernel that takes all rows, in torch here, a step's projection is what calling it gives."""
    model = Mamba3(64, depth=1)
    mixer = model.layers[0].mixer
    taken = []

    def linear(x, weight, residual=None, **norm):
        taken.append(weight)
        y = torch.nn.functional.linear(x, weight)
        return y if residual is None else residual + y

    def step_projection(proj, mixer, cache, inplace):
        return proj[:, 0, :mixer.d_inner].unflatten(-1, (mixer.nheads, mixer.headdim)), cache

    monkeypatch.setattr(ops, "linear_supported", lambda x, weight: True)
    monkeypatch.setattr(ops, "linear", linear)
    monkeypatch.setattr(ops, "step_projection", step_projection)
    if change is not None:
        change(mixer, name)
    x = torch.randn(3, 1, 64)
    with torch.no_grad():
        got, _ = mixer.step(x, None, residual=x)
        mixed = step_projection(mixer.in_proj(x), mixer, None, False)[0].flatten(-2)
        want = x + mixer.out_proj(mixed).unsqueeze(1)
    # (the same products in other orders: a row of in_proj adds 64, one of out_proj 128 of them)
    assert torch.allclose(got, want, rtol=0, atol=256 * 2.0 ** -24 * (want.abs().max().item() + 128))
    assert len(taken) == (2 if change is None else 1)


def _stubs(monkeypatch):
    """The kernels of a step in torch, enough of them for a step off the GPU: the caches count their steps."""

    def step_projection(proj, mixer, cache, inplace):
        assert inplace
        for t in cache:
            t += 1
        return torch.zeros(proj.shape[0], mixer.nheads, mixer.headdim, dtype=proj.dtype), cache

    def rms_norm8(x, weight, eps, *, add=None, keep_sum=False):
        return ops.Rows8(torch.zeros(x.shape, dtype=torch.int8), torch.ones(x.shape[:-1])), x if keep_sum else None

    def linear8(rows, weight, residual=None, *, out=None, dtype=None):
        return torch.zeros(*rows.shape[:-1], weight.shape[0], dtype=dtype)

    monkeypatch.setattr(ops, "step_projection", step_projection)
    monkeypatch.setattr(ops, "rms_norm8", rms_norm8)
    monkeypatch.setattr(ops, "linear8", linear8)
    monkeypatch.setattr(ops, "quantize8_rows", lambda x: rms_norm8(x, None, 0.0)[0])


@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("name", ["in_proj", "out_proj"])
@pytest.mark.parametrize("maker,rows", [("quantize_prefill", 65), ("quantize_decode", 65), ("quantize_decode", 2)])
def test_a_refused_step_moves_no_cache(monkeypatch, maker, rows, name, layer):
    """A stale copy anywhere is refused before the first layer's cache is updated in place."""
    _stubs(monkeypatch)
    model = Mamba3(64, depth=2).to(BF16)
    x = torch.zeros(rows, 1, 64, dtype=BF16)
    cache = [block.mixer.allocate_cache(rows, device=x.device, dtype=BF16) for block in model.layers]
    copies = (lambda: model.quantize_decode(32)) if maker == "quantize_decode" else model.quantize_prefill
    copies()
    with torch.no_grad():
        model.step(x, cache, inplace=True)
        assert all((t == 1).all() for states in cache for t in states)
        getattr(model.layers[layer].mixer, name).weight.mul_(2)
        with pytest.raises(RuntimeError, match=f"{name}.weight changed since {maker}"):
            model.step(x, cache, inplace=True)
        assert all((t == 1).all() for states in cache for t in states)
        mixer, states = model.layers[layer].mixer, cache[layer]
        with pytest.raises(RuntimeError, match=f"{name}.weight changed since {maker}"):
            mixer.step(x, states, inplace=True)
        assert all((t == 1).all() for t in states)
        copies()
        model.step(x, cache, inplace=True)
        assert all((t == 2).all() for states in cache for t in states)


def test_few_rows_do_not_ask_for_8_bits(monkeypatch):
    """Steps of up to 64 rows run on the weights as they are, also on changed ones."""
    _stubs(monkeypatch)
    model = Mamba3(64, depth=2).to(BF16).quantize_prefill()
    with torch.no_grad():
        model.layers[1].mixer.out_proj.weight.mul_(2)
        cache = [block.mixer.allocate_cache(64, device=torch.device("cpu"), dtype=BF16) for block in model.layers]
        model.step(torch.zeros(64, 1, 64, dtype=BF16), cache, inplace=True)
    assert all((t == 1).all() for states in cache for t in states)


class _OwnMixer(torch.nn.Module):
    """A mixer of someone's own in a layer's place: what it has to take is what it always had to."""

    def forward(self, hidden_states, return_cache=False):
        return (2 * hidden_states, None) if return_cache else 2 * hidden_states

    def step(self, hidden_states, cache, *, inplace=False, residual=None, norm=None):
        y = 2 * (hidden_states if norm is None else norm(hidden_states))
        return y if residual is None else residual + y, cache


@pytest.mark.parametrize("call", [lambda m, x: m(x), lambda m, x: m.prefill(x)[0], lambda m, x: m.step(x)[0],
                                  lambda m, x: m.step(x[:2])[0]])
def test_mixers_of_one_s_own(call):
    model = Mamba3(64, depth=2)
    for layer in model.layers:
        layer.mixer = _OwnMixer()
    x = torch.randn(70, 1, 64)
    with torch.no_grad():
        got = call(model, x)
        h = x[:got.shape[0]]
        for layer in model.layers:
            h = h + 2 * layer.norm(h)
        assert torch.equal(got, model.norm_f(h))
