"""``m3_gated_scan`` / ``m3_gated_scan_bwd`` (``ops.gated_scan``, ``ops.gated_step``) against the
recurrence in 64 bits, token by token (``oracle/gated.py``).

The bounds are the oracle's running error bounds of an FP32 evaluation on the same inputs, plus
half a step of the output's type (2^-8 of the value for bf16, 2^-11 for f16, 2^-24 for FP32; f16
also half its smallest step, 2^-25). Gradients are compared with torch's own differentiation of the 64-bit
recurrence, and once with differences of the kernel's outputs.
"""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import _hip, ops
from oracle import gated as og

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _inputs(batch, length, width, dtype, form, seed=0, sliced=False, state=False, lengths=False,
            reset=False, spread=1.0):
    g = torch.Generator().manual_seed(1000 * seed + 31 * batch + 7 * length + width)

    def rand(*shape):
        return torch.randn(*shape, generator=g)

    if sliced:  # columns of one projection's output, as the layer has them
        proj = (spread * rand(batch, length, 3 * width + 5)).to(dtype)
        x, decay, gate = (proj[..., i * width:(i + 1) * width] for i in range(3))
    else:
        x, decay, gate = ((spread * rand(batch, length, width)).to(dtype) for _ in range(3))
    rate = None
    if form == "gate":
        rate = torch.exp(1.5 * rand(width) - 2)
    else:
        gate = None
        decay = (-torch.exp(rand(batch, length, width) - 2)).to(dtype)
    out = dict(x=x, decay=decay, gate=gate, rate=rate,
               state=rand(batch, width) if state else None, lengths=None, reset=None)
    if lengths:
        n = torch.randint(0, length + 1, (batch,), generator=g, dtype=torch.int32)
        n[0] = length + 3 if batch > 1 else n[0]   # past the end: clamped
        n[-1] = 0 if batch > 2 else n[-1]          # a row with no token
        out["lengths"] = n
    if reset:
        out["reset"] = torch.rand(batch, length, generator=g) < 0.05
        out["reset"][0, 0] = True
        if length > 3:
            out["reset"][-1, 1:3] = True           # two in a row
    return out


def _to(case, **kw):
    return {k: None if v is None else v.to(DEV) for k, v in case.items()}


def _call(c):
    return ops.gated_scan(c["x"], c["decay"], c["gate"], c["rate"], initial_state=c["state"],
                          lengths=c["lengths"], reset=c["reset"])


def _near(name, got, want, bound, dtype):
    got = got.detach().double().cpu()
    limit = bound + HALF[dtype] * (want.abs() + bound) + (2.0 ** -25 if dtype == F16 else 1e-37)
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = ((got - want).abs() / limit).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: error / bound = {worst:.3f}"


SHAPES = [(1, 1, 1), (2, 1, 7), (3, 5, 64), (2, 16, 130), (2, 127, 66), (2, 128, 128), (1, 129, 256),
          (3, 300, 33), (2, 513, 130), (1, 1100, 70)]


@pytest.mark.parametrize("options", ["plain", "sliced", "state", "lengths", "reset", "all"])
@pytest.mark.parametrize("form", ["gate", "given"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype, form, options):
    on = {o: options in (o, "all") for o in ("sliced", "state", "lengths", "reset")}
    case = _inputs(*shape, dtype, form, **on)
    want, final = og.scan(**case)
    bound = og.bounds(**case)
    # slices are made on the GPU's copy of the whole projection, so that strides survive
    c = _to(case)
    if on["sliced"]:
        base = case["x"]._base.to(DEV)
        w = shape[2]
        c["x"], c["decay"] = base[..., :w], base[..., w:2 * w]
        c["decay"] = c["decay"] if form == "gate" else case["decay"].to(DEV)
        c["gate"] = base[..., 2 * w:3 * w] if form == "gate" else None
    with torch.inference_mode():
        y, last = _call(c)
    assert y.dtype == dtype and last.dtype == F32
    _near("y", y, want, bound["y"], dtype)
    _near("final", last, final, bound["final"], F32)


@pytest.mark.parametrize("options", ["plain", "state", "lengths", "reset", "all"])
@pytest.mark.parametrize("form", ["gate", "given"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(shape, dtype, form, options):
    on = {o: options in (o, "all") for o in ("state", "lengths", "reset")}
    case = _inputs(*shape, dtype, form, seed=1, **on)
    g = torch.Generator().manual_seed(5)
    dy = torch.randn(shape, generator=g).to(dtype)
    dfinal = torch.randn(shape[0], shape[2], generator=g)
    names = [n for n in ("x", "decay", "gate", "rate", "state") if case[n] is not None]
    wide = dict(case)
    for n in names:
        wide[n] = case[n].double().requires_grad_(True)
    y64, f64 = og.scan(**wide)
    want = torch.autograd.grad((y64, f64), [wide[n] for n in names], (dy.double(), dfinal.double()))
    bound = og.bounds(**case, dy=dy, dfinal=dfinal)
    c = _to(case)
    for n in names:
        c[n].requires_grad_(True)
    y, last = _call(c)
    got = torch.autograd.grad((y, last), [c[n] for n in names], (dy.to(DEV), dfinal.to(DEV)))
    _near("y", y, y64.detach(), bound["y"], dtype)
    for n, a, b in zip(names, got, want):
        assert a.dtype == c[n].dtype
        _near("d" + n, a, b, bound["d" + n], a.dtype)


def test_gradients_against_differences():
    """The kernel's gradients along a random direction of every input, against central
    differences of its own FP32 outputs. The loss weighs outputs with FP32 numbers and sums them
    in 64 bits; a step of 2^-7 leaves a cubic term of relative size 2^-14, the rounding of the
    outputs (2^-24 of about 1 each, 4,000 of them) about 2^-24 * 64 * 64 = 2^-12 over the step: 2^-5 absolute
    at most, against a directional derivative of the order of sqrt(4,000) = 64."""
    case = _to(_inputs(2, 40, 50, F32, "gate", seed=3, state=True, reset=True))
    names = ("x", "decay", "gate", "rate", "state")
    g = torch.Generator().manual_seed(2)
    wy = torch.randn(2, 40, 50, generator=g).to(DEV).double()
    wf = torch.randn(2, 50, generator=g).to(DEV).double()
    way = {n: torch.randn(case[n].shape, generator=g).to(DEV) for n in names}
    way["rate"] = way["rate"] * case["rate"] * 0.2

    def loss(step):
        c = dict(case)
        for n in names:
            c[n] = case[n] + step * way[n]
        with torch.no_grad():
            y, last = _call(c)
        return ((y.double() * wy).sum() + (last.double() * wf).sum()).item()

    h = 2.0 ** -7
    c = dict(case)
    for n in names:
        c[n] = case[n].clone().requires_grad_(True)
    y, last = _call(c)
    grads = torch.autograd.grad((y, last), [c[n] for n in names], (wy.float(), wf.float()))
    slope = sum((a.double() * way[n].double()).sum().item() for n, a in zip(names, grads))
    change = (loss(h) - loss(-h)) / (2 * h)
    size = sum((a.double() * way[n].double()).abs().sum().item() for n, a in zip(names, grads))
    assert abs(slope - change) <= 2.0 ** -5 + 2.0 ** -12 * size


@pytest.mark.parametrize("backward", [False, True])
def test_masked_places_may_hold_anything(backward):
    """NaN and infinities past a row's end, and before a reset, reach nothing else."""
    case = _inputs(3, 200, 70, F32, "gate", seed=4, state=True)
    case["lengths"] = torch.tensor([150, 0, 200], dtype=torch.int64)
    case["reset"] = torch.zeros(3, 200, dtype=torch.bool)
    case["reset"][2, 140] = True
    clean = _to(case)
    dirty = {k: None if v is None else v.clone() for k, v in clean.items()}
    for n, bad in (("x", float("nan")), ("decay", float("inf")), ("gate", float("nan"))):
        dirty[n][0, 150:] = bad
        dirty[n][1] = bad
    dirty["x"][2, 17] = float("nan")
    dirty["x"][2, 90, 3] = float("inf")
    dy = torch.randn(3, 200, 70, device=DEV)
    dy_dirty = dy.clone()
    dy_dirty[0, 150:] = float("nan")
    names = ("x", "decay", "gate", "state") if backward else ()
    results = []
    for c, d in ((clean, dy), (dirty, dy_dirty)):
        for n in names:
            c[n].requires_grad_(True)
        y, last = _call(c)
        grads = torch.autograd.grad((y, last), [c[n] for n in names],
                                    (d, torch.ones_like(last))) if backward else ()
        results.append((y.detach(), last.detach(), *grads))
    for a, b in zip(*results):
        assert torch.equal(a[:2], b[:2])           # rows 0 and 1: the padding
        if a.dim() == 3:
            assert torch.equal(a[2, 140:], b[2, 140:])  # row 2 from the reset on
    y, last = results[1][:2]
    assert torch.equal(last[2], results[0][1][2])
    assert torch.equal(last[1], clean["state"][1]) and not y[1].any() and not y[0, 150:].any()
    assert torch.isnan(y[2, 17:140]).all()


@pytest.mark.parametrize("form", ["gate", "given"])
def test_extreme_logits(form):
    """Gates fully shut and fully open, rates of 0 and beyond exp's range: values of the
    recurrence's limits, no NaN."""
    logits = torch.tensor([-200.0, -100.0, -30.0, 0.0, 30.0, 100.0, float("-inf"), float("inf")])
    width = logits.numel() * 4
    x = torch.ones(1, 3, width)
    decay = logits.repeat(4).expand(1, 3, width).contiguous()
    gate = rate = None
    if form == "gate":
        gate = torch.ones(1, 3, width)
        rate = torch.tensor([0.0, 1e-30, 1.0, 1e30]).repeat_interleave(logits.numel())
    else:
        decay = torch.minimum(decay, torch.tensor(0.0))
    c = _to(dict(x=x, decay=decay, gate=gate, rate=rate, state=torch.full((1, width), 2.0),
                 lengths=None, reset=None))
    for n in ("x", "decay", "gate", "rate"):
        if c[n] is not None:
            c[n].requires_grad_(True)
    y, last = _call(c)
    leaves = [c[n] for n in ("x", "decay", "gate", "rate") if c[n] is not None]
    grads = torch.autograd.grad(y.sum(), leaves)
    a = torch.exp(-rate.double() * torch.sigmoid(decay.double())) if form == "gate" else \
        torch.exp(decay.double())
    w = torch.sqrt(-torch.expm1(2 * -rate.double() * torch.sigmoid(decay.double()))) * \
        torch.sigmoid(torch.ones((), dtype=torch.float64)) if form == "gate" else 1.0
    h = torch.full((1, width), 2.0, dtype=torch.float64)
    for t in range(3):
        h = a[:, t] * h + (w[:, t] if form == "gate" else 1.0)
        # factors of at least 2^-126 or taken as 0: the bound is a few steps of FP32
        torch.testing.assert_close(y[:, t].double().cpu(), h, rtol=2e-6, atol=1e-30)
    for grad in grads:
        assert torch.isfinite(grad).all()


@pytest.mark.parametrize("form", ["gate", "given"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("batch,width", [(1, 1), (1, 4096), (5, 333), (64, 512), (256, 130)])
def test_step(batch, width, dtype, form):
    case = _inputs(batch, 1, width, dtype, form, seed=6, state=True)
    want, final = og.scan(**case)
    bound = og.bounds(**case)
    c = _to(case)
    gate = None if c["gate"] is None else c["gate"][:, 0]
    state = c["state"].clone()
    with torch.inference_mode():
        y, new = ops.gated_step(c["x"][:, 0], c["decay"][:, 0], state, gate, c["rate"])
        assert torch.equal(state, c["state"])
        y2, same = ops.gated_step(c["x"][:, 0], c["decay"][:, 0], state, gate, c["rate"],
                                  inplace=True)
    assert same is state and torch.equal(state, new) and torch.equal(y, y2)
    _near("y", y.unsqueeze(1), want, bound["y"], dtype)
    _near("state", new, final, bound["final"], F32)


def test_steps_continue_a_scan():
    """Prefill of a padded batch, then tokens one at a time: the sequence scanned whole."""
    batch, width, lengths = 4, 200, [5, 131, 260, 0]
    case = _to(_inputs(batch, 270, width, F32, "gate", seed=7))
    n = torch.tensor(lengths, dtype=torch.int32)
    with torch.inference_mode():
        _, state = ops.gated_scan(case["x"], case["decay"], case["gate"], case["rate"],
                                  lengths=n.to(DEV))
        rows = torch.arange(batch, device=DEV)
        for i in range(6):
            at = n.to(DEV).long() + i
            _, state = ops.gated_step(case["x"][rows, at], case["decay"][rows, at], state,
                                      case["gate"][rows, at], case["rate"])
    whole = {k: None if v is None else v.cpu() for k, v in case.items()}
    whole["lengths"] = n + 6
    _, want = og.scan(**whole)
    _near("state", state, want, 2 * og.bounds(**whole)["final"], F32)


def test_offsets_past_32_bits():
    """Rows more than 2^31 elements apart, tokens 16,384."""
    width, length = 96, 140
    far = (1 << 31) + 64
    buffer = torch.zeros(far + length * 16384 + width, dtype=BF16, device=DEV)
    view = buffer.as_strided((2, length, width), (far, 16384, 1))
    case = _inputs(2, length, width, BF16, "given", seed=8)
    view.copy_(case["x"].to(DEV))
    c = _to(case)
    with torch.inference_mode():
        want = _call(c)
        got = _call(c | dict(x=view))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_expanded_and_transposed_inputs():
    """A decay shared by all tokens (stride 0), x with another axis innermost, a summed loss
    (whose gradient is one number, expanded)."""
    case = _to(_inputs(2, 150, 64, F32, "gate", seed=9))
    decay = case["decay"][:, :1]
    x = case["x"].transpose(1, 2).contiguous().transpose(1, 2)
    leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_(True)
              for t in (x, decay, case["gate"], case["rate"])]
    y, _ = ops.gated_scan(leaves[0], leaves[1].expand(2, 150, 64), leaves[2], leaves[3])
    y.sum().backward()
    plain = [t.detach().contiguous().requires_grad_(True) for t in leaves]
    wide = plain[1].expand(2, 150, 64).contiguous()
    y2, _ = ops.gated_scan(plain[0], wide, plain[2], plain[3])
    torch.autograd.backward(y2, torch.ones_like(y2))
    assert torch.equal(y, y2)
    for a, b in zip(leaves, plain):
        assert torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("length", [1, 5, 20, 128, 129, 700])
def test_the_final_state_is_the_last_token_s_and_may_lie_on_the_first(length):
    """FP32: final_state equals out at each row's last token bit for bit, also where the C call is
    given the initial state's memory for it."""
    case = _to(_inputs(3, length, 70, F32, "gate", seed=16, state=True))
    n = torch.tensor([length, max(1, length // 2), 0], device=DEV, dtype=torch.int32)
    with torch.inference_mode():
        y, last = _call(case | dict(lengths=n))
        for b, k in enumerate(n.tolist()):
            assert torch.equal(last[b], y[b, k - 1] if k else case["state"][b])
        out, state = torch.empty_like(y), case["state"].clone()
        values = (*ops._gated_inputs(case["x"], case["decay"], case["gate"], case["rate"], state, n,
                                     None), *ops._packed(out), *ops._packed(state), *(0,) * 8)
        size = _hip.need("m3_gated_scan_workspace_size", _hip.GATED_SCAN.pack(*values, 0, 0))
        ws = torch.empty(size + 1, dtype=torch.uint8, device=DEV)
        _hip.launch("m3_gated_scan", _hip.GATED_SCAN.pack(*values, ws.data_ptr(), size), y.device.index)
        assert torch.equal(state, last) and torch.equal(out, y)


def test_repeated_calls_agree_bit_for_bit():
    case = _to(_inputs(2, 3000, 130, BF16, "gate", seed=10))
    dy = torch.randn(2, 3000, 130, device=DEV).to(BF16)
    leaves = [case[n].requires_grad_(True) for n in ("x", "decay", "gate", "rate")]
    first = None
    for _ in range(4):
        y, last = _call(case)
        got = (y.detach(), last.detach(), *torch.autograd.grad(y, leaves, dy))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_streams_and_graphs():
    """Calls on two streams at once, and forward with gradients captured and replayed between
    eager calls, give what one call alone gives."""
    cases = [_to(_inputs(2, 700, 130, BF16, "gate", seed=s)) for s in (11, 12)]
    dy = torch.randn(2, 700, 130, device=DEV).to(BF16)

    def both(c):
        leaves = [c[n].detach().requires_grad_(True) for n in ("x", "decay", "gate", "rate")]
        y, last = ops.gated_scan(*leaves)
        return [y.detach(), last.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = [[t.clone() for t in both(c)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = both(cases[i])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs = []
    for c in cases:
        static = {k: None if v is None else v.clone() for k, v in c.items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both(static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = both(static)
        graphs.append((graph, static, outs))
    for turn in range(4):
        for i, (graph, static, outs) in enumerate(graphs):
            other = (i + turn) % 2
            for n in ("x", "decay", "gate", "rate"):
                static[n].copy_(cases[other][n])
            graph.replay()
            eager = both(cases[other])
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs, want[other]))
            assert all(torch.equal(x, y) for x, y in zip(eager, want[other]))


@pytest.mark.parametrize("length", [1, 40, 500])
def test_a_loss_on_one_output(length):
    """A loss on the final state alone, or on the outputs alone: the other's gradient is zeros."""
    case = _to(_inputs(2, length, 66, BF16, "gate", seed=13, state=True))
    names = ("x", "decay", "gate", "rate", "state")
    for n in names:
        case[n].requires_grad_(True)
    leaves = [case[n] for n in names]
    y, last = _call(case)
    zero_y, zero_last = torch.zeros_like(y), torch.zeros_like(last)
    weigh_y, weigh_last = torch.randn_like(y), torch.randn_like(last)
    alone = torch.autograd.grad((y * weigh_y).sum(), leaves, retain_graph=True)
    both = torch.autograd.grad((y, last), leaves, (weigh_y, zero_last), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(alone, both))
    alone = torch.autograd.grad((last * weigh_last).sum(), leaves, retain_graph=True)
    both = torch.autograd.grad((y, last), leaves, (zero_y, weigh_last))
    assert all(torch.equal(a, b) for a, b in zip(alone, both))


def test_a_rate_and_a_state_shared_by_broadcast():
    """A 16-bit rate, one number for all channels, and one state for all rows: their gradients are
    the sums over what they were broadcast to."""
    case = _to(_inputs(3, 90, 50, F32, "gate", seed=14))
    rate = torch.full((1,), 0.25, device=DEV, dtype=BF16, requires_grad=True)
    state = torch.randn(1, 50, device=DEV, requires_grad=True)
    y, last = ops.gated_scan(case["x"], case["decay"], case["gate"], rate.expand(50),
                             initial_state=state.expand(3, 50))
    y.sum().backward()
    wide_rate = torch.full((50,), 0.25, device=DEV, requires_grad=True)
    wide_state = state.detach().expand(3, 50).contiguous().requires_grad_(True)
    y2, _ = ops.gated_scan(case["x"], case["decay"], case["gate"], wide_rate,
                           initial_state=wide_state)
    torch.autograd.backward(y2, torch.ones_like(y2))
    assert torch.equal(y, y2)
    # sums of 50 and 3 terms in FP32, the first rounded to bf16
    total = wide_rate.grad.double().sum()
    size = wide_rate.grad.double().abs().sum()
    assert (rate.grad.double() - total).abs() <= 2.0 ** -8 * total.abs() + 50 * 2.0 ** -24 * size \
        + 2.0 ** -8 * size
    torch.testing.assert_close(state.grad, wide_state.grad.sum(0, keepdim=True), rtol=1e-6, atol=1e-6)


def test_lengths_beyond_32_bits_and_below_zero():
    case = _to(_inputs(4, 300, 34, F32, "given", seed=15))
    with torch.inference_mode():
        want = ops.gated_scan(case["x"], case["decay"],
                              lengths=torch.tensor([300, 0, 7, 300], device=DEV))
        for n in (torch.tensor([1 << 40, -(1 << 40), 7, 301], device=DEV),
                  torch.tensor([2 ** 31 - 1, -2 ** 31, 7, 301], device=DEV, dtype=torch.int32)):
            got = ops.gated_scan(case["x"], case["decay"], lengths=n)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_many_narrow_rows_and_too_many():
    """One channel, 100,000 rows; and more tiles than a grid holds, refused."""
    x = torch.randn(100_000, 20, 1, device=DEV)
    decay = -torch.rand(100_000, 20, 1, device=DEV)
    with torch.inference_mode():
        y, last = ops.gated_scan(x, decay)
        h = torch.zeros(100_000, 1, device=DEV, dtype=torch.float64)
        for t in range(20):
            h = torch.exp(decay[:, t].double()) * h + x[:, t]
            # 20 tokens, each off by less than 2^-20 of sums of at most 20 values below 6
            assert (y[:, t] - h).abs().max().item() <= 20 * 2.0 ** -20 * 6 * 20
        assert torch.equal(last, y[:, -1])
        few = torch.zeros(1, 1, 1, device=DEV, dtype=BF16)
        with pytest.raises(RuntimeError, match="2\\^23 tiles"):
            ops.gated_scan(few.expand(1 << 23, 17, 1), few.expand(1 << 23, 17, 1))


def test_empty_extents():
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = torch.randn(shape, device=DEV)
        state = torch.randn(shape[0], shape[2], device=DEV)
        y, last = ops.gated_scan(x, x, initial_state=state)
        assert y.shape == x.shape and torch.equal(last, state)
        assert not ops.gated_scan(x, x)[1].any()
    x = torch.randn(0, 8, device=DEV)
    assert ops.gated_step(x, x, x)[0].shape == (0, 8)


def test_empty_extents_under_autograd_and_another_default_type():
    x = torch.randn(2, 0, 8, device=DEV, requires_grad=True)
    torch.set_default_dtype(F16)
    try:
        y, last = ops.gated_scan(x, x)
    finally:
        torch.set_default_dtype(F32)
    assert last.dtype == F32 and last.shape == (2, 8)
    (y.sum() + last.sum()).backward()
    assert x.grad.shape == x.shape


def test_second_derivatives_are_refused():
    x, decay = (torch.randn(1, 4, 8, device=DEV, requires_grad=True) for _ in range(2))
    y, _ = ops.gated_scan(x, decay)
    grad, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), x)
    state = torch.zeros(1, 8, device=DEV)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.gated_step(x[:, 0], decay[:, 0], state)


@pytest.mark.parametrize("length,width", [(1, 6), (12, 7), (60, 66), (200, 33), (300, 130)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_reset_token_s_own_decay_reaches_nothing(length, width, dtype):
    """Given form: what stands in decay at a reset token, infinite, NaN or above exp's range, changes
    neither outputs nor gradients, and its own gradient is 0."""
    case = _inputs(3, length, width, dtype, "given", seed=17, state=True)
    case["reset"] = torch.zeros(3, length, dtype=torch.bool)
    case["reset"][0, 0] = case["reset"][1, length // 2] = case["reset"][2, length - 1] = True
    g = torch.Generator().manual_seed(6)
    dy = torch.randn(3, length, width, generator=g).to(dtype).to(DEV)
    dfinal = torch.randn(3, width, generator=g).to(DEV)
    names, first = ("x", "decay", "state"), None
    for value in (-0.5, 0.0, 100.0, float("inf"), float("nan"), float("-inf")):
        c = _to(case)
        c["decay"][c["reset"]] = value
        for n in names:
            c[n].requires_grad_(True)
        y, last = _call(c)
        got = (y.detach(), last.detach(),
               *torch.autograd.grad((y, last), [c[n] for n in names], (dy, dfinal)))
        assert not got[3][c["reset"]].any()
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("level", [8.0, 12.0, 17.0, 24.0])
def test_gradients_of_saturated_gates(dtype, level):
    """Logits far out, to both sides: the complement of a sigmoid keeps its digits (in f16 the incoming
    gradient is large, so that the results are not below its range). The 64-bit side forms 1 - p
    from p, whose sum 1 + e^-x rounds by up to 2^-53 and quotient by 2^-54: below 2^-52, (1 + e^|x|) 2^-52 of it."""
    case = _inputs(2, 70, 40, dtype, "gate", seed=18, state=True)
    g = torch.Generator().manual_seed(7)
    for n in ("decay", "gate"):
        side = torch.where(torch.rand(2, 70, 40, generator=g) < 0.5, -1.0, 1.0)
        case[n] = (side * level * (1 + 0.1 * torch.rand(2, 70, 40, generator=g))).to(dtype)
    big = 2.0 ** 12 if dtype == F16 else 1.0
    dy = (big * torch.randn(2, 70, 40, generator=g)).to(dtype)
    dfinal = big * torch.randn(2, 40, generator=g)
    names = ("x", "decay", "gate", "rate", "state")
    wide = {n: v if n not in names else v.double().requires_grad_(True) for n, v in case.items()}
    y64, f64 = og.scan(**wide)
    want = torch.autograd.grad((y64, f64), [wide[n] for n in names], (dy.double(), dfinal.double()))
    bound = og.bounds(**case, dy=dy, dfinal=dfinal)
    for n, v in zip(names, want):
        if n in ("decay", "gate"):
            bound["d" + n] += 2.0 ** -52 * (1 + case[n].double().abs().exp()) * v.abs()
    c = _to(case)
    for n in names:
        c[n].requires_grad_(True)
    y, last = _call(c)
    got = torch.autograd.grad((y, last), [c[n] for n in names], (dy.to(DEV), dfinal.to(DEV)))
    for n, a, b in zip(names, got, want):
        inside = b.abs() < (65504 if a.dtype == F16 else 3e38)
        _near("d" + n, torch.where(inside, a.detach().double().cpu(), 0), torch.where(inside, b, 0),
              bound["d" + n], a.dtype)


# many workgroups: (batch, length, width) of over 2,048 tiles of 128 tokens (one counter for all
# chains), over 2,048 of 64 only (the backward's alone), and few chains of over 64 links (the look-back's
# window), with pairs of channels and single ones
LONG = [(64, 4300, 6), (33, 8500, 7), (40, 3400, 10), (1, 8500, 130), (2, 9000, 33)]


def _long(shape, dtype, form, **on):
    """Channels that remember thousands of tokens, so that a wrong carry between tiles shows."""
    case = _inputs(*shape, dtype, form, seed=19, **on)
    if form == "gate":
        case["rate"] = case["rate"] * 0.02
    else:
        case["decay"] = (case["decay"].float() * 0.02).to(dtype)
    if case["reset"] is not None:
        g = torch.Generator().manual_seed(8)
        case["reset"] = torch.rand(shape[:2], generator=g) < 1e-3
    return case


@pytest.mark.parametrize("shape,dtype,form,options", [
    *[(s, BF16, "gate", "all") for s in LONG],
    *[(s, d, f, "all") for s, d, f in zip(LONG, (F32, F16, F32, F16, F32), ("gate", "given") * 3)],
    (LONG[0], BF16, "given", "plain"), (LONG[3], BF16, "gate", "plain"), (LONG[4], F32, "given", "plain")])
def test_many_and_long_chains(shape, dtype, form, options):
    """Outputs and gradients in 64 bits, token by token; two calls on two streams at once agree."""
    case = _long(shape, dtype, form, **{o: options == "all" for o in ("state", "lengths", "reset")})
    g = torch.Generator().manual_seed(9)
    dy = torch.randn(shape, generator=g).to(dtype)
    dfinal = torch.randn(shape[0], shape[2], generator=g)
    names = [n for n in ("x", "decay", "gate", "rate", "state") if case[n] is not None]
    wide = {n: v if n not in names else v.double().requires_grad_(True) for n, v in case.items()}
    y64, f64 = og.scan(**wide)
    want = torch.autograd.grad((y64, f64), [wide[n] for n in names], (dy.double(), dfinal.double()))
    bound = og.bounds(**case, dy=dy, dfinal=dfinal)
    c, dy, dfinal = _to(case), dy.to(DEV), dfinal.to(DEV)
    torch.cuda.synchronize()
    results = []
    for stream in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(stream):
            leaves = {n: c[n].detach().requires_grad_(True) for n in names}
            y, last = _call(c | leaves)
            results.append((y.detach(), last.detach(),
                            *torch.autograd.grad((y, last), list(leaves.values()), (dy, dfinal))))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))
    y, last, *got = results[0]
    _near("y", y, y64.detach(), bound["y"], dtype)
    _near("final", last, f64.detach(), bound["final"], F32)
    for n, a, b in zip(names, got, want):
        _near("d" + n, a, b, bound["d" + n], a.dtype)


def test_a_state_updated_in_place_is_not_lost_on_autograd():
    """A backward pass over an initial state that a step has since overwritten, or over an input
    that a product has, is refused as torch refuses its own in-place writes."""
    case = _to(_inputs(2, 30, 32, BF16, "gate", seed=20, state=True))
    token = [case[n][:, 0].clone() for n in ("x", "decay", "gate")]
    case["rate"].requires_grad_(True)
    y, _ = _call(case)
    with torch.no_grad():
        ops.gated_step(token[0], token[1], case["state"], token[2], case["rate"].detach(), inplace=True)
    with pytest.raises(RuntimeError, match="inplace"):
        y.float().sum().backward()
    wide = torch.randn(32, 32, device=DEV).to(BF16)
    weight = ops.quantize4(wide, 32)
    for product, w in ((ops.linear4, weight), (ops.linear, wide)):
        x = torch.randn(2, 1, 32, device=DEV).to(BF16)
        y, _ = ops.gated_scan(x, case["decay"][:, :1], case["gate"][:, :1], case["rate"])
        with torch.no_grad():
            product(token[0], w, out=x[:, 0])
        with pytest.raises(RuntimeError, match="inplace"):
            y.float().sum().backward()
    with torch.inference_mode():  # tensors without versions are written all the same
        state, out = torch.zeros(2, 32, device=DEV), torch.empty(2, 32, device=DEV, dtype=BF16)
        assert ops.gated_step(*token[:2], state, inplace=True)[1] is state
        assert ops.linear4(token[0], weight, out=out) is out


def test_tokens_far_apart():
    """Rows of one token far apart, and a gradient whose tokens are: as their contiguous copies."""
    far = (1 << 24) + 8
    case = _to(_inputs(2, 3, 32, BF16, "gate", seed=21))
    buffer = torch.zeros(3 * far, device=DEV, dtype=BF16)
    for n in ("x", "decay"):
        view = buffer.as_strided((2, 3, 32), (64, far, 1), 0 if n == "x" else 128)
        view.copy_(case[n])
        case[n + "_far"] = view
    x, decay = (case[n].requires_grad_(True) for n in ("x", "decay"))
    dy = torch.randn(2, 3, 32, device=DEV).to(BF16)
    dy_far = buffer.as_strided((2, 3, 32), (64, far, 1), 256)
    dy_far.copy_(dy)
    y, _ = ops.gated_scan(x, decay, case["gate"], case["rate"])
    want = torch.autograd.grad(y, (x, decay), dy, retain_graph=True)
    got = torch.autograd.grad(y, (x, decay), dy_far)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        assert torch.equal(ops.gated_scan(case["x_far"], case["decay_far"], case["gate"],
                                          case["rate"])[0], y)
        one = ops.gated_scan(case["x_far"][:1, :1], case["decay_far"][:1, :1], case["gate"][:1, :1],
                             case["rate"])[0]
        assert torch.equal(one, y[:1, :1])


@pytest.mark.parametrize("shape", [(2, 0, 8), (0, 5, 8), (2, 5, 0)])
def test_gradients_without_tokens(shape):
    """Every input that asks for a gradient gets one: the final state's for the initial one, else zeros."""
    x, decay, gate = (torch.randn(shape, device=DEV, requires_grad=True) for _ in range(3))
    rate = torch.rand(shape[2], device=DEV, requires_grad=True)
    state = torch.randn(shape[0], shape[2], device=DEV, requires_grad=True)
    y, last = ops.gated_scan(x, decay, gate, rate, initial_state=state)
    assert torch.equal(last, state) and y.shape == x.shape
    weigh = torch.randn_like(last)
    grads = torch.autograd.grad((y, last), (x, decay, gate, rate, state), (torch.zeros_like(y), weigh))
    for grad, t in zip(grads, (x, decay, gate, rate, state)):
        assert grad.shape == t.shape and grad.dtype == t.dtype
    assert not grads[3].any() and (shape[1] > 0 or torch.equal(grads[4], weigh))
    y, _ = ops.gated_scan(x, decay, gate, rate, initial_state=state)
    assert not torch.autograd.grad(y.sum(), state)[0].any()
