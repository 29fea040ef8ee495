"""The 8-bit projections' operators, as they are measured: the residual stream's RMSNorm with rows of 8
bits as its output (``ops.rms_norm8``), rows rounded to 8 bits (``ops.quantize8_rows``), and the
product of such rows with a weight in 8 bits (``ops.linear8``), one by one and in the order in which
a block calls them.

``listed()`` holds the fixed cases and ``draw(rng)`` makes further ones of the same ranges.
``prepare`` builds what a program has in hand before a call, ``run`` makes one pass (in plain torch,
or with ``own`` through the package's entry points), ``work`` states the bytes and operations the
pass cannot do without, and ``exact`` computes the same outputs in 64 bits.

Rows in 8 bits: a row p (x, or its sum with the residual times the norm's weight) has codes
``rint(127 p / max|p|)``, ties to even, of the exact quotient, and one scale; they come back as the
values ``code * scale``.
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
        # one token of one user between two blocks: latency only
        dict(name="norm8_b1", kind="norm8", rows=1, inner=2048, dtype="bf16", add="bf16"),
        # the residual stream of a prefilled batch under autocast: FP32 rows, 16-bit mixer output
        dict(name="norm8_prefill", kind="norm8", rows=65536, inner=1024, dtype="f32", add="bf16"),
        # a short prompt's rows of odd width, at odd alignments
        dict(name="rows8_odd", kind="rows8", rows=777, inner=1111, dtype="f16"),
        # a prefilled batch's mixer outputs before out_proj
        dict(name="rows8_prefill", kind="rows8", rows=32768, inner=4096, dtype="bf16"),
        # in_proj of one token of one user: the weight's stream and latency
        dict(name="linear8_b1", kind="linear8", rows=1, inner=2048, outer=8672, dtype="bf16",
             residual=False),
        # out_proj of a small decode batch, the residual added
        dict(name="linear8_b16", kind="linear8", rows=16, inner=4096, outer=2048, dtype="f16",
             residual=True),
        # in_proj of a full decode batch
        dict(name="linear8_b256", kind="linear8", rows=256, inner=2048, outer=8672, dtype="bf16",
             residual=False),
        # a small layer over a ragged prompt: no size a multiple of a tile's, FP32 out
        dict(name="linear8_odd", kind="linear8", rows=333, inner=1111, outer=1217, dtype="f32",
             residual=True),
        # in_proj of a prefilled batch at the benchmark's width: much is written for what is computed
        dict(name="linear8_prefill", kind="linear8", rows=65536, inner=1024, outer=4480,
             dtype="bf16", residual=False),
        # a wide projection over a long prompt: bound by what is computed
        dict(name="linear8_wide", kind="linear8", rows=8192, inner=8192, outer=28672,
             dtype="bf16", residual=False),
        # a block's way into its mixer: residual add, norm, rounding, in_proj
        dict(name="block_in", kind="block_in", rows=16384, inner=2048, outer=8672, dtype="bf16",
             add="bf16"),
        # and out of it: rounding, out_proj
        dict(name="block_out", kind="block_out", rows=4000, inner=4096, outer=2048, dtype="bf16",
             residual=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Columns: mostly whole vectors, some odd."""
    width = _log(rng, lo, hi)
    return width if rng.random() < 0.3 else max(8, width // 8 * 8)


def draw(rng):
    kind = rng.choice(["norm8", "rows8", "linear8", "linear8", "linear8", "block_in", "block_out"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    inner = _width(rng, 32, 8192)
    rows = min(_log(rng, 1, 65536), (1 << 27) // inner)
    case = dict(kind=kind, rows=rows, inner=inner, dtype=dtype)
    if kind in ("norm8", "block_in"):
        case["add"] = rng.choice([dtype, dtype, "none"] + (["bf16", "f16"] if dtype == "f32" else []))
    if kind in ("norm8", "rows8"):
        return case
    outer = _width(rng, 16, 28672)
    most = min(1 << 27, (1 << 40) // inner)
    case["rows"] = max(1, min(rows, most // outer))
    case["outer"] = outer
    if kind != "block_in":
        case["residual"] = rng.random() < 0.4
    return case


# --------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    state = dict(case=case)
    rows, inner, dtype = case["rows"], case["inner"], DTYPES[case["dtype"]]
    if case["kind"] == "linear8":
        # rows of normal values in 8 bits: 127 lies at about four standard deviations
        state["codes"] = (32 * rand(rows, inner)).round_().clamp_(-127, 127).to(torch.int8)
        state["scales"] = (0.5 + torch.rand(rows, generator=g, device=DEVICE)) / 32
    else:
        state["x"] = rand(rows, inner).to(dtype)
    if case["kind"] in ("norm8", "block_in"):
        state["add"] = None
        if case["add"] != "none":
            state["add"] = (0.3 * rand(rows, inner)).to(DTYPES[case["add"]])
        state["norm"] = 1 + 0.1 * rand(inner)
    if "outer" in case:
        outer = case["outer"]
        state["w_codes"] = (32 * rand(outer, inner)).round_().clamp_(-127, 127).to(torch.int8)
        scale = 0.5 + torch.rand(outer, generator=g, device=DEVICE)
        state["w_scales"] = scale / (32 * math.sqrt(inner))
        state["residual"] = rand(rows, outer).to(dtype) if case.get("residual") else None
        if own:
            from mamba3_amd import ops

            state["weight"] = ops.Weight8(state["w_codes"], state["w_scales"])
    return state


# --------------------------------------------------------------------------- plain forms


def _plain_sum(s):
    """The residual stream's rows: x, or x + add rounded to x's type."""
    if s["add"] is None:
        return s["x"]
    return (s["x"].float() + s["add"].float()).to(s["x"].dtype)


def _plain_codes(p, factor):
    """Rows p in 64 bits -> their codes, and scales in FP32 that hold `factor` too. Whether a value
    lies below or above half a code needs more than 32 bits."""
    most = p.abs().amax(-1, keepdim=True)
    codes = torch.where(most > 0, torch.round(127 * p / most), 0.0)
    return codes.float(), most.float() * factor / 127


def _plain_rows8(x):
    return _plain_codes(x.double(), 1.0)


def _plain_norm8(s):
    total = _plain_sum(s)
    wide = total.float()
    rms = torch.rsqrt(wide.square().mean(-1, keepdim=True) + EPS)
    weight = s["norm"].to(total.dtype)
    return *_plain_codes(total.double() * weight.double(), rms), total


def _plain_product(s, codes, scales):
    out = codes @ s["w_codes"].float().t()
    out = out * (scales * s["w_scales"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(DTYPES[s["case"]["dtype"]])


def _plain_run(s):
    kind = s["case"]["kind"]
    if kind == "linear8":
        return _plain_product(s, s["codes"].float(), s["scales"].unsqueeze(1))
    if kind in ("rows8", "block_out"):
        codes, scales = _plain_rows8(s["x"])
        return codes * scales if kind == "rows8" else _plain_product(s, codes, scales)
    codes, scales, total = _plain_norm8(s)
    out = codes * scales if kind == "norm8" else _plain_product(s, codes, scales)
    return (out, total) if s["add"] is not None else out


# --------------------------------------------------------------------------- the package's calls


def _own_run(s):
    from mamba3_amd import ops

    kind, dtype = s["case"]["kind"], DTYPES[s["case"]["dtype"]]
    if kind == "linear8":
        rows = ops.Rows8(s["codes"], s["scales"])
        return ops.linear8(rows, s["weight"], s["residual"], dtype=dtype)
    if kind in ("rows8", "block_out"):
        rows = ops.quantize8_rows(s["x"])
        if kind == "rows8":
            return rows.dequantize()
        return ops.linear8(rows, s["weight"], s["residual"], dtype=dtype)
    rows, total = ops.rms_norm8(s["x"], s["norm"], EPS, add=s["add"], keep_sum=s["add"] is not None)
    out = rows.dequantize() if kind == "norm8" else ops.linear8(rows, s["weight"], dtype=dtype)
    return out if total is None else (out, total)


def run(state):
    if own:
        return _own_run(state)
    return _plain_run(state)


# --------------------------------------------------------------------------- needed work


def work(case):
    rows, inner, size = case["rows"], case["inner"], SIZE[case["dtype"]]
    elements = rows * inner
    if case["kind"] == "linear8":
        bytes_, flops = elements + rows * 4, 0
    else:
        bytes_, flops = elements * size, 3 * elements
    if case["kind"] in ("norm8", "block_in"):
        flops += 4 * elements
        bytes_ += inner * 4
        if case["add"] != "none":
            bytes_ += elements * (SIZE[case["add"]] + size)
    if case["kind"] in ("norm8", "rows8"):
        return dict(bytes=bytes_ + elements * 4, flops=flops)
    outer = case["outer"]
    bytes_ += outer * (inner + 4) + rows * outer * size * (2 if case.get("residual") else 1)
    return dict(bytes=bytes_, flops=flops + 2 * elements * outer)


# --------------------------------------------------------------------------- 64 bits


def _exact_rows(p):
    """The values that a row's codes stand for, with the scale of p: by quotient and remainder."""
    most = p.abs().max(dim=1, keepdim=True).values
    part = 127 * p.abs()
    whole = torch.floor(part / most)
    twice = 2 * (part - whole * most)
    up = (twice > most) | ((twice == most) & (whole % 2 == 1))
    values = torch.sign(p) * (whole + up) * (most / 127)
    return torch.where(most > 0, values, torch.zeros_like(p))


def exact(case, seed):
    s = prepare(case, seed)
    total = None
    if case["kind"] == "linear8":
        values = s["codes"].double() * s["scales"].double().unsqueeze(1)
    elif case["kind"] in ("rows8", "block_out"):
        values = _exact_rows(s["x"].double())
    else:
        rows = s["x"]
        if s["add"] is not None:
            # the stream is held in its type: the sum is rounded to it, for the norm as well
            rows = total = (rows.double() + s["add"].double()).to(rows.dtype)
        rows = rows.double()
        mean = rows.pow(2).sum(1, keepdim=True) / case["inner"]
        weight = s["norm"].to(s["x"].dtype).double()
        values = _exact_rows(rows * weight) / (mean + EPS).sqrt()
    if "outer" in case:
        values = values @ s["w_codes"].double().t().contiguous() * s["w_scales"].double()
        if s["residual"] is not None:
            values = values + s["residual"].double()
    return values if total is None else (values, total.double())
