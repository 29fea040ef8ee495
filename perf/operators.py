"""The recurrent layer's operators, as they are measured: the gated linear recurrence over a sequence
(``ops.gated_scan``, forward and with its gradients), its single token (``ops.gated_step``) and
the projections of a few rows with 4-bit weights (``ops.linear4``).

``listed()`` holds the fixed cases and ``draw(rng)`` makes further ones of the same ranges.
``prepare`` builds what a program has in hand before a call, ``run`` makes one pass (in plain torch,
or with ``own`` through the package's entry points), ``work`` states the bytes and operations the
pass cannot do without, and ``exact`` computes the same outputs in 64 bits, token by token.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5


def listed():
    return [
        # one token of one user: a layer's state of 4096 channels, latency only
        dict(name="step_b1", kind="step", batch=1, width=4096, dtype="bf16", form="gate"),
        # one token of a full serving batch
        dict(name="step_b256", kind="step", batch=256, width=4096, dtype="f16", form="gate"),
        # one user's prompt of ordinary, ragged length before decoding at batch 1
        dict(name="prompt_b1", kind="scan", batch=1, length=1777, width=4096, dtype="bf16",
             form="gate", lengths=False, reset=False, state=False),
        # prefill of a served batch: prompts of unequal lengths, padded at the end
        dict(name="prefill_padded", kind="scan", batch=8, length=8192, width=2048, dtype="bf16",
             form="gate", lengths=True, reset=False, state=False),
        # one long row of packed documents, each beginning from an empty state
        dict(name="long_packed", kind="scan", batch=1, length=65536, width=1536, dtype="bf16",
             form="gate", lengths=False, reset=True, state=True),
        # log decays given, FP32, odd sizes
        dict(name="given_f32", kind="scan", batch=3, length=1023, width=250, dtype="f32",
             form="given", lengths=False, reset=False, state=True),
        # a training step's pass through the recurrence, ordinary size
        dict(name="train_batch", kind="train", batch=8, length=4096, width=2048, dtype="bf16",
             form="gate", lengths=False, reset=False, state=False),
        # training in FP32 at odd sizes, packed rows, a state carried in
        dict(name="train_f32", kind="train", batch=5, length=777, width=333, dtype="f32",
             form="gate", lengths=False, reset=True, state=True),
        # in_proj of a decode step at batch 1, the block's norm fused
        dict(name="in_proj_b1", kind="linear4", rows=1, inner=2048, outer=8672, group=128,
             dtype="bf16", zeros=False, norm=True, residual=False),
        # out_proj of a decode step at batch 16, the residual add fused
        dict(name="out_proj_b16", kind="linear4", rows=16, inner=4096, outer=2048, group=64,
             dtype="f16", zeros=True, norm=False, residual=True),
        # a small layer at an odd batch, fine groups, odd output width
        dict(name="odd_b5", kind="linear4", rows=5, inner=1120, outer=1111, group=32,
             dtype="bf16", zeros=True, norm=False, residual=False),
        # a wide projection at batch 64
        dict(name="wide_b64", kind="linear4", rows=64, inner=8192, outer=28672, group=128,
             dtype="bf16", zeros=False, norm=False, residual=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    """Channels: mostly whole vectors, some odd."""
    width = _log(rng, 64, 4096)
    return width if rng.random() < 0.3 else max(8, width // 8 * 8)


def draw(rng):
    kind = rng.choice(["step", "scan", "scan", "scan", "train", "train", "linear4", "linear4",
                       "linear4"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    form = rng.choice(["gate", "gate", "given"])
    if kind == "step":
        return dict(kind=kind, batch=_log(rng, 1, 256), width=_width(rng), dtype=dtype, form=form)
    if kind in ("scan", "train"):
        width, length = _width(rng), _log(rng, 1, 65536)
        most = (1 << 26) // (4 if dtype == "f32" else 1) // (2 if kind == "train" else 1)
        batch = _log(rng, 1, max(1, min(64, most // (width * length))))
        length = max(1, min(length, most // (batch * width)))
        return dict(kind=kind, batch=batch, length=length, width=width, dtype=dtype, form=form,
                    lengths=rng.random() < 0.4, reset=rng.random() < 0.3,
                    state=rng.random() < 0.5)
    group = rng.choice([32, 64, 128, 128])
    inner = max(1, _log(rng, 256, 8192) // group) * group
    return dict(kind=kind, rows=_log(rng, 1, 64), inner=inner, outer=_log(rng, 64, 28672),
                group=group, dtype=rng.choice(["bf16", "bf16", "f16"]),
                zeros=rng.random() < 0.5, norm=rng.random() < 0.3, residual=rng.random() < 0.3)


# --------------------------------------------------------------------------- inputs


def _recurrence_inputs(case, g, lead):
    """x, decay, gate as a layer's projection gives them (slices of its output), and the rate."""
    width, dtype = case["width"], DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if case["form"] == "gate":
        if case["kind"] == "train":
            x, decay, gate = (rand(*lead, width).to(dtype) for _ in range(3))
        else:
            proj = rand(*lead, 3 * width).to(dtype)
            x, decay, gate = proj.split(width, dim=-1)
        # a channel keeps 0.9 to 0.999 of its state a token where its gate is fully open
        rate = -8.0 * torch.log(0.9 + 0.099 * torch.rand(width, generator=g, device=DEVICE))
        return x, decay, gate, rate
    x = rand(*lead, width).to(dtype)
    decay = (-torch.exp(1.5 * rand(*lead, width) - 3.0)).to(dtype)  # log decays, mostly -0.01 to -1
    return x, decay, None, None


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case=case)
    if case["kind"] == "linear4":
        rows, inner, outer, group = case["rows"], case["inner"], case["outer"], case["group"]
        dtype = DTYPES[case["dtype"]]
        state["x"] = torch.randn(rows, inner, generator=g, device=DEVICE).to(dtype)
        state["packed"] = torch.randint(0, 256, (outer, inner // 2), generator=g, device=DEVICE,
                                        dtype=torch.uint8)
        scale = 0.5 + torch.rand(outer, inner // group, generator=g, device=DEVICE)
        state["scales"] = (scale / (4.6 * math.sqrt(inner))).to(dtype)
        state["zeros"] = state["norm"] = state["residual"] = None
        if case["zeros"]:
            state["zeros"] = torch.randint(5, 11, (outer, inner // group), generator=g,
                                           device=DEVICE, dtype=torch.uint8)
        if case["norm"]:
            weight = 1 + 0.1 * torch.randn(inner, generator=g, device=DEVICE)
            state["norm"] = weight.to(dtype)
        if case["residual"]:
            state["residual"] = torch.randn(rows, outer, generator=g, device=DEVICE).to(dtype)
        if own:
            from mamba3_amd import ops

            state["weight"] = ops.Weight4(state["packed"], state["scales"], state["zeros"])
        return state
    batch, width = case["batch"], case["width"]
    if case["kind"] == "step":
        state["x"], state["decay"], state["gate"], state["rate"] = _recurrence_inputs(
            case, g, (batch,))
        state["state"] = torch.randn(batch, width, generator=g, device=DEVICE)
        return state
    length = case["length"]
    state["x"], state["decay"], state["gate"], state["rate"] = _recurrence_inputs(
        case, g, (batch, length))
    state["lengths"] = state["reset"] = state["state"] = None
    if case["lengths"]:
        state["lengths"] = torch.randint(max(1, length // 2), length + 1, (batch,), generator=g,
                                         device=DEVICE, dtype=torch.int32)
    if case["reset"]:
        # documents of 500 tokens on average
        state["reset"] = torch.rand(batch, length, generator=g, device=DEVICE) < 0.002
    if case["state"]:
        state["state"] = torch.randn(batch, width, generator=g, device=DEVICE)
    if case["kind"] == "train":
        state["dy"] = torch.randn(batch, length, width, generator=g,
                                  device=DEVICE).to(DTYPES[case["dtype"]])
        state["dfinal"] = torch.randn(batch, width, generator=g, device=DEVICE)
        for name in ("x", "decay", "gate", "rate", "state"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# --------------------------------------------------------------------------- plain forms


def _plain_coefficients(s):
    """FP32 log decay, input weight sqrt(1 - a^2) (None: 1) and the two gates' sigmoids."""
    decay = s["decay"].detach().float()
    if s["gate"] is None:
        return decay, None, None, None
    open_r = torch.sigmoid(decay)
    open_g = torch.sigmoid(s["gate"].detach().float())
    log_a = -s["rate"].detach() * open_r
    return log_a, torch.sqrt(-torch.expm1(2 * log_a)), open_r, open_g


def _plain_scan(a, b):
    """Every prefix of h <- a h + b along dim 1, by doubling: spans of 1, 2, 4, ... tokens."""
    span, length = 1, a.shape[1]
    while span < length:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], dim=1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], dim=1)
        span *= 2
    return b


def _plain_past_end(s, length):
    if s["lengths"] is None:
        return None
    at = torch.arange(length, device=DEVICE)
    return (at >= s["lengths"].unsqueeze(1)).unsqueeze(-1)


def _plain_forward(s):
    x = s["x"].detach().float()
    log_a, weight, open_r, open_g = _plain_coefficients(s)
    carry = torch.exp(log_a)
    if s["reset"] is not None:
        carry = torch.where(s["reset"].unsqueeze(-1), 0.0, carry)
    b = x if weight is None else weight * open_g * x
    past = _plain_past_end(s, x.shape[1])
    if past is not None:
        carry, b = torch.where(past, 1.0, carry), torch.where(past, 0.0, b)
    if s["state"] is not None:
        first = b[:, :1] + carry[:, :1] * s["state"].detach().unsqueeze(1)
        h = _plain_scan(carry, torch.cat([first, b[:, 1:]], dim=1))
    else:
        h = _plain_scan(carry, b)
    return h, carry, past, (log_a, weight, open_r, open_g, x)


def _plain_run_scan(s):
    h, _, past, _ = _plain_forward(s)
    y = h if past is None else torch.where(past, 0.0, h)
    return y.to(s["x"].dtype), h[:, -1].clone()


def _plain_run_train(s):
    h, carry, past, (log_a, weight, open_r, open_g, x) = _plain_forward(s)
    y = h if past is None else torch.where(past, 0.0, h)
    dy = s["dy"].float()
    if past is not None:
        dy = torch.where(past, 0.0, dy)
    # D_t = dy_t + carry_{t+1} D_{t+1}, the final state's gradient joining at the last token
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dfinal"].unsqueeze(1)], dim=1)
    after = torch.cat([carry[:, 1:], torch.zeros_like(carry[:, :1])], dim=1)
    d = _plain_scan(after.flip(1), dy.flip(1)).flip(1)
    before = torch.zeros_like(h[:, :1]) if s["state"] is None else s["state"].detach().unsqueeze(1)
    before = torch.cat([before, h[:, :-1]], dim=1)
    dstate = carry[:, 0] * d[:, 0]
    dlog = d * carry * before
    if past is not None:
        d, dlog = torch.where(past, 0.0, d), torch.where(past, 0.0, dlog)
    dtype = s["x"].dtype
    out = dict(y=y.to(dtype), final=h[:, -1].clone())
    if s["state"] is not None:
        out["dstate"] = dstate
    if weight is None:
        return out | dict(dx=d.to(dtype), ddecay=dlog.to(dtype))
    slope = torch.where(weight > 0, torch.exp(2 * log_a) / weight, 0.0)
    dlog = dlog - d * open_g * x * slope
    return out | dict(
        dx=(d * weight * open_g).to(dtype),
        ddecay=(dlog * -s["rate"].detach() * open_r * (1 - open_r)).to(dtype),
        dgate=(d * weight * x * open_g * (1 - open_g)).to(dtype),
        drate=-(dlog * open_r).double().sum((0, 1)).float())


def _plain_run_step(s):
    log_a, weight, _, open_g = _plain_coefficients(s)
    x = s["x"].float()
    b = x if weight is None else weight * open_g * x
    state = torch.exp(log_a) * s["state"] + b
    return state.to(s["x"].dtype), state


def _codes(packed):
    """[N, K / 2] bytes -> [N, K] codes: the low four bits are the even column."""
    return torch.stack([packed & 15, packed >> 4], dim=-1).flatten(1)


def _plain_run_linear4(s):
    case = s["case"]
    shape = (case["outer"], -1, case["group"])
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().unsqueeze(-1)
    weight = (_codes(s["packed"]).float().view(shape) - zeros) * s["scales"].float().unsqueeze(-1)
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["norm"].float()
    out = x @ weight.flatten(1).t()
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(s["x"].dtype)


_PLAIN = dict(scan=_plain_run_scan, train=_plain_run_train, step=_plain_run_step,
              linear4=_plain_run_linear4)


# --------------------------------------------------------------------------- the package's calls


def _own_run(s):
    from mamba3_amd import ops

    kind = s["case"]["kind"]
    if kind == "linear4":
        return ops.linear4(s["x"], s["weight"], s["residual"], norm_weight=s["norm"], norm_eps=EPS)
    if kind == "step":
        return ops.gated_step(s["x"], s["decay"], s["state"], s["gate"], s["rate"])
    y, final = ops.gated_scan(s["x"], s["decay"], s["gate"], s["rate"], initial_state=s["state"],
                              lengths=s["lengths"], reset=s["reset"])
    if kind == "scan":
        return y, final
    names = [n for n in ("x", "decay", "gate", "rate", "state") if s[n] is not None]
    grads = torch.autograd.grad((y, final), [s[n] for n in names], (s["dy"], s["dfinal"]))
    return dict(y=y, final=final) | {"d" + n: d for n, d in zip(names, grads)}


def run(state):
    if own:
        return _own_run(state)
    return _PLAIN[state["case"]["kind"]](state)


# --------------------------------------------------------------------------- needed work


def work(case):
    if case["kind"] == "linear4":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        groups = outer * inner // case["group"]
        size = SIZE[case["dtype"]]
        return dict(bytes=outer * inner // 2 + groups * (size + int(case["zeros"]))
                    + rows * (inner + outer) * size
                    + (rows * outer * size if case["residual"] else 0)
                    + (inner * size if case["norm"] else 0),
                    flops=2 * rows * inner * outer)
    size, arrays = SIZE[case["dtype"]], 3 if case["form"] == "gate" else 2
    states = case["batch"] * case["width"] * 4
    elements = case["batch"] * case["width"] * case.get("length", 1)
    # tokens past a row's length (a quarter of them on average) are written, not read
    read = 0.75 if case.get("lengths") else 1.0
    ops_each = 20 if case["form"] == "gate" else 4
    bytes_ = elements * size * (arrays * read + 1) + states * (1 + int(bool(case.get("state", 1))))
    if case.get("reset"):
        bytes_ += case["batch"] * case["length"]
    if case["kind"] == "train":
        bytes_ += elements * size * ((arrays + 1) * read + arrays)
        bytes_ += states * (1 + 2 * int(case["state"]))
        ops_each *= 3
    return dict(bytes=int(bytes_), flops=int(elements * ops_each * read))


# --------------------------------------------------------------------------- 64 bits


def _exact_coefficients(s):
    decay = s["decay"].detach().double()
    if s["gate"] is None:
        return decay, torch.ones_like(decay)
    log_a = s["rate"].detach().double().neg() / (1 + torch.exp(-decay))
    return log_a, (1 - torch.exp(2 * log_a)).sqrt() / (1 + torch.exp(-s["gate"].detach().double()))


def _exact_linear4(s, case):
    low, high = (s["packed"] & 15).double(), (s["packed"] >> 4).double()
    group = case["group"] // 2
    zeros = torch.full_like(s["scales"], 8.0) if s["zeros"] is None else s["zeros"]
    zeros = zeros.double().repeat_interleave(group, 1)
    scales = s["scales"].double().repeat_interleave(group, 1)
    x = s["x"].double()
    if s["norm"] is not None:
        x = x / (x.pow(2).sum(1, keepdim=True) / case["inner"] + EPS).sqrt() * s["norm"].double()
    out = x[:, 0::2] @ ((low - zeros) * scales).t().contiguous()
    out += x[:, 1::2] @ ((high - zeros) * scales).t().contiguous()
    return out if s["residual"] is None else out + s["residual"].double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear4":
        return _exact_linear4(s, case)
    log_a, weight = _exact_coefficients(s)
    x = s["x"].detach().double()
    if case["kind"] == "step":
        h = torch.exp(log_a) * s["state"].double() + weight * x
        return h, h.clone()
    batch, length, width = x.shape
    carry, b = torch.exp(log_a), weight * x
    if s["reset"] is not None:
        carry = carry * (~s["reset"]).unsqueeze(-1)
    valid = torch.ones(batch, length, 1, dtype=torch.bool, device=DEVICE)
    if s["lengths"] is not None:
        valid = (torch.arange(length, device=DEVICE) < s["lengths"].unsqueeze(1)).unsqueeze(-1)
        carry, b = torch.where(valid, carry, 1.0), b * valid
    h = torch.zeros(batch, width, dtype=torch.float64, device=DEVICE)
    if s["state"] is not None:
        h = h + s["state"].detach()
    before = torch.empty_like(b)  # the state each token finds
    after = torch.empty_like(b)  # the state each token leaves
    for t in range(length):
        before[:, t] = h
        h = torch.addcmul(b[:, t], carry[:, t], h)
        after[:, t] = h
    if case["kind"] == "scan":
        return after * valid, h
    out = dict(y=after * valid, final=h)
    dy = s["dy"].double() * valid
    d = after  # reused: the gradient of each token's state
    grad = s["dfinal"].double()
    for t in range(length - 1, -1, -1):
        grad = grad + dy[:, t]
        d[:, t] = grad
        grad = grad * carry[:, t]
    if case["state"]:
        out["dstate"] = grad
    dlog = d * carry * before * valid
    d = d * valid
    if s["gate"] is None:
        return out | dict(dx=d, ddecay=dlog)
    rate = s["rate"].detach().double()
    p = torch.sigmoid(s["decay"].detach().double())
    q = torch.sigmoid(s["gate"].detach().double())
    root = (1 - torch.exp(2 * log_a)).sqrt()
    dlog = dlog - d * q * x * torch.exp(2 * log_a) / root
    return out | dict(dx=d * weight, ddecay=-dlog * rate * p * (1 - p),
                      dgate=d * weight * x * (1 - q), drate=-(dlog * p).sum((0, 1)))
