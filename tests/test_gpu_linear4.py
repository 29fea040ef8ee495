"""``m3_linear4`` (``ops.linear4``, ``ops.Weight4``) against the product in 64 bits.

Bound per element, from the kernel's arithmetic: half a step of the output's type, and FP32
sums. A group's share is scale * (16 A - (16 + z) X) with A = sum (1 + q / 16) x, X = sum x: at most 62
scale |x| a column (31 and 31), summed over at most 128 columns and then over the groups and waves,
each sum off by 2^-24 of the terms' absolute sum: (128 + K / group + 40) 2^-24 * 62 sum |x| scale.
With the norm the operand x * w is rounded to 16 bits (half a step of each term) and the factor
1 / rms is off by a few steps of FP32.
"""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import Mamba3, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F16 = torch.bfloat16, torch.float16
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _weight(n, k, group, scale_dtype, zeros, g):
    packed = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(n, k // group, generator=g)) / (4.6 * k ** 0.5)).to(scale_dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1).double().view(n, -1, group)
    shift = 8.0 if z is None else z.double().unsqueeze(-1)
    wide = ((codes - shift) * scales.double().unsqueeze(-1)).flatten(1)
    return packed, scales, z, wide


def _check(got, x, wide, scales, group, residual=None, norm=None, eps=1e-5):
    k = x.shape[1]
    xd, extra = x.double().cpu(), 0.0
    if norm is not None:
        rms = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
        xd = xd * norm.to(x.dtype).double().cpu() * rms
        extra = (HALF[x.dtype] + 2.0 ** -20) * (xd.abs() @ wide.abs().t())
        if x.dtype == F16:  # products below f16's normal range: half its smallest step
            extra = extra + 2.0 ** -25 * rms * wide.abs().sum(1)
    want = xd @ wide.t()
    if residual is not None:
        want = want + residual.double().cpu()
    full = scales.double().cpu().repeat_interleave(group, 1)
    bound = (128 + k // group + 40) * 2.0 ** -24 * 62 * (xd.abs() @ full.t()) + extra
    limit = bound + HALF[x.dtype] * (want.abs() + bound) + (2.0 ** -25 if x.dtype == F16 else 1e-37)
    worst = ((got.double().cpu() - want).abs() / limit).max().item()
    assert worst <= 1.0, f"error / bound = {worst:.3f}"


SHAPES = [(1, 1, 32), (1, 17, 128), (2, 100, 160), (5, 1111, 1120), (15, 64, 256), (16, 2048, 1024),
          (17, 33, 384), (31, 48, 2048), (33, 260, 512), (48, 130, 96), (64, 512, 4096),
          (65, 40, 128), (130, 100, 256), (256, 31, 640)]


@pytest.mark.parametrize("options", ["plain", "zeros", "residual", "norm", "all"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear4(shape, dtype, group, options):
    m, n, k = shape
    if k % group:
        with pytest.raises(ValueError, match="multiple of group"):
            ops.quantize4(torch.zeros(n, k, dtype=dtype), group)
        return
    g = torch.Generator().manual_seed(m + 7 * n + k)
    zeros, residual, norm = (options in (o, "all") for o in ("zeros", "residual", "norm"))
    # scales in the other 16-bit type for some
    scale_dtype = dtype if m % 2 else (F16 if dtype == BF16 else BF16)
    packed, scales, z, wide = _weight(n, k, group, scale_dtype, zeros, g)
    x = torch.randn(m, k, generator=g).to(dtype)
    res = torch.randn(m, n, generator=g).to(dtype) if residual else None
    nw = 1 + 0.1 * torch.randn(k, generator=g) if norm else None
    dev = [None if t is None else t.to(DEV) for t in (packed, scales, z, x, res, nw)]
    weight = ops.Weight4(*dev[:3])
    with torch.inference_mode():
        got = ops.linear4(dev[3], weight, dev[4], norm_weight=dev[5])
    _check(got, x, wide, scales, group, res, nw)


@pytest.mark.parametrize("m,n,k", [(1, 28672, 8192), (64, 28672, 1024), (1, 64, 65536)])
def test_large(m, n, k):
    g = torch.Generator().manual_seed(k)
    packed, scales, z, wide = _weight(n, k, 128, BF16, True, g)
    x = torch.randn(m, k, generator=g).to(BF16)
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV))
    with torch.inference_mode():
        got = ops.linear4(x.to(DEV), weight)
    _check(got, x, wide, scales, 128)


def test_one_column_at_a_time():
    """A unit x reads one column: every code of the weight comes back exactly."""
    g = torch.Generator().manual_seed(0)
    for group in (32, 64, 128):
        packed, _, z, _ = _weight(50, 384, group, BF16, True, g)
        scales = torch.full((50, 384 // group), 0.5, dtype=BF16)
        weight = ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV))
        want = weight.dequantize(torch.float32)
        eye = torch.eye(384, dtype=F16, device=DEV)
        with torch.inference_mode():
            got = torch.cat([ops.linear4(eye[i:i + 128], weight) for i in range(0, 384, 128)])
        assert torch.equal(got.float().t(), want)


def test_strided_and_unaligned_operands():
    """Rows that are slices, at odd offsets; out with rows further apart; out as the residual."""
    g = torch.Generator().manual_seed(1)
    m, n, k = 9, 70, 256
    packed, scales, z, wide = _weight(n, k, 64, BF16, True, g)
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV))
    base = torch.randn(m, k + 21, generator=g).to(BF16)
    wide_out = torch.full((m, n + 13), 7.0, dtype=BF16, device=DEV)
    with torch.inference_mode():
        x = base.to(DEV)[:, 3:3 + k]
        ops.linear4(x, weight, out=wide_out[:, 5:5 + n])
        _check(wide_out[:, 5:5 + n], base[:, 3:3 + k], wide, scales, 64)
        assert (wide_out[:, :5] == 7).all() and (wide_out[:, 5 + n:] == 7).all()
        res = torch.randn(m, n, generator=g).to(BF16)
        both = res.to(DEV)
        ops.linear4(x, weight, both, out=both)
        _check(both, base[:, 3:3 + k], wide, scales, 64, res)
        turned = x.t().contiguous().t()
        assert torch.equal(ops.linear4(turned, weight), ops.linear4(x, weight))
        unaligned = torch.ones(k + 1, device=DEV, dtype=BF16)[1:]
        assert torch.equal(ops.linear4(x, weight, norm_weight=unaligned),
                           ops.linear4(x, weight, norm_weight=unaligned.clone()))


def test_rows_do_not_touch_each_other():
    """A row of NaN or infinities spoils its own outputs only, a bad scale its own column."""
    g = torch.Generator().manual_seed(2)
    packed, scales, z, _ = _weight(64, 512, 128, BF16, True, g)
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV))
    x = torch.randn(20, 512, generator=g).to(BF16).to(DEV)
    bad = x.clone()
    bad[3], bad[17, 5] = float("nan"), float("inf")
    with torch.inference_mode():
        for norm in (None, torch.ones(512, device=DEV, dtype=BF16)):
            want = ops.linear4(x, weight, norm_weight=norm)
            got = ops.linear4(bad, weight, norm_weight=norm)
            keep = [i for i in range(20) if i not in (3, 17)]
            assert torch.equal(got[keep], want[keep])
            assert torch.isnan(got[3]).all()
        scales[9, 1] = float("nan")
        spoilt = ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV))
        got, want = ops.linear4(x, spoilt), ops.linear4(x, weight)
        keep = [i for i in range(64) if i != 9]
        assert torch.isnan(got[:, 9]).all() and torch.equal(got[:, keep], want[:, keep])


@pytest.mark.parametrize("m,n,k,group", [(40, 6200, 256, 128), (64, 6145, 1184, 32), (33, 9000, 448, 64),
                                         (64, 16400, 384, 128), (200, 6144, 128, 64),
                                         (100, 24576, 128, 32), (64, 12304, 2048, 128)])
def test_many_rows_of_both(m, n, k, group):
    """The shapes on which a workgroup stages x once (from 384 tile rows, above 16 rows of x): one
    and two tile rows a wave, one and two teams, odd counts of tiles, columns that end inside a tile."""
    g = torch.Generator().manual_seed(n)
    packed, scales, z, wide = _weight(n, k, group, BF16, n % 2 == 0, g)
    x = torch.randn(m, k, generator=g).to(BF16)
    res = torch.randn(m, n, generator=g).to(BF16)
    nw = 1 + 0.1 * torch.randn(k, generator=g)
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV), None if z is None else z.to(DEV))
    bad = x.to(DEV).clone()
    bad[m // 2] = float("nan")
    with torch.inference_mode():
        _check(ops.linear4(x.to(DEV), weight), x, wide, scales, group)
        _check(ops.linear4(x.to(DEV), weight, res.to(DEV), norm_weight=nw.to(DEV)), x, wide, scales,
               group, res, nw)
        want, got = ops.linear4(x.to(DEV), weight), ops.linear4(bad, weight)
    keep = [i for i in range(m) if i != m // 2]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[m // 2]).all()


def test_streams_and_graph():
    g = torch.Generator().manual_seed(3)
    packed, scales, z, _ = _weight(200, 1024, 128, BF16, False, g)
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV))
    xs = [torch.randn(4, 1024, generator=g).to(BF16).to(DEV) for _ in range(2)]
    with torch.inference_mode():
        want = [ops.linear4(x, weight) for x in xs]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in xs], [None, None]
        for _ in range(5):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i] = ops.linear4(xs[i], weight)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        static = xs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear4(static, weight)
        for i in (0, 1, 1, 0):
            static.copy_(xs[i])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]) and torch.equal(ops.linear4(xs[i], weight), want[i])


@pytest.mark.parametrize("batch", [1, 5, 40, 70])
@pytest.mark.parametrize("rank", [1, 4])
def test_quantized_decode_matches_the_dequantized_model(batch, rank):
    """``quantize_decode``: steps (4-bit weights up to 64 rows) against the same model's steps through its
    16-bit weights, which hold the same values rounded once. Both paths round the projections'
    outputs to bf16 and differ by the weights' rounding (2^-9) and one rounding of each
    intermediate; four layers of either agree to 2% of the output's scale."""
    torch.manual_seed(0)
    model = Mamba3(256, d_state=128, depth=4, mimo_rank=rank).eval().to(DEV, BF16)
    model.quantize_decode(64)
    plain = Mamba3(256, d_state=128, depth=4, mimo_rank=rank).eval().to(DEV, BF16)
    plain.load_state_dict(model.state_dict())
    calls = []
    real = ops.linear4
    try:
        ops.linear4 = lambda *a, **k: calls.append(1) or real(*a, **k)
        with torch.inference_mode():
            x = torch.randn(batch, 20, 256, device=DEV).to(BF16)
            got, cache = model.prefill(x)
            want, cache2 = plain.prefill(x)
            assert torch.equal(got, want) and not calls
            for _ in range(3):
                x = torch.randn(batch, 1, 256, device=DEV).to(BF16)
                got, cache = model.step(x, cache)
                want, cache2 = plain.step(x, cache2)
                scale = want.float().abs().max().item()
                assert (got - want).float().abs().max().item() <= 2e-2 * scale
    finally:
        ops.linear4 = real
    assert len(calls) == (3 * 2 * 4 if batch <= ops.DECODE_LINEAR_ROWS else 0)


def test_quantized_decode_in_a_graph_and_after_changes():
    torch.manual_seed(1)
    model = Mamba3(256, d_state=128, depth=2).eval().to(DEV, BF16).quantize_decode()
    decoder = model.cuda_graph(batch_size=2)
    with torch.inference_mode():
        cache = None
        for _ in range(4):
            x = torch.randn(2, 1, 256, device=DEV).to(BF16)
            want, cache = model.step(x, cache)
            assert torch.equal(decoder(x, validate=True), want)
        model.layers[0].mixer.in_proj.weight.data = model.layers[0].mixer.in_proj.weight.data.clone()
        with pytest.raises(RuntimeError, match="quantize_decode"):
            model.step(x, cache)
        with pytest.raises(RuntimeError, match="recreate"):
            decoder(x, validate=True)
        model.quantize_decode()
        model.step(x, cache)


@pytest.mark.parametrize("width,length", [(256, 40), (512, 300)])
def test_a_recurrent_layer_from_the_operators(width, length):
    """A layer as the operators are used together: the norm and in_proj in 4 bits, the gated
    recurrence, out_proj in 4 bits with the residual. Prefill of a padded batch (dequantised
    products, the scan), then tokens by ``linear4`` and ``gated_step``, against the layer in 64 bits
    over the whole sequence. The layer rounds to bf16 four times (projection, recurrence, output
    and, in prefill, the normed rows): 2^-8 of values of the outputs' scale each, with sums of 256 or more
    terms behind the first: 4 * 2^-8 * 2 of the scale."""
    from oracle import gated as og
    g = torch.Generator().manual_seed(width)
    norm = (1 + 0.1 * torch.randn(width, generator=g)).to(BF16)
    w_in = (torch.randn(3 * width, width, generator=g) / width ** 0.5).to(BF16)
    w_out = (torch.randn(width, width, generator=g) / width ** 0.5).to(BF16)
    rate = torch.rand(width, generator=g) + 0.05
    lengths = torch.tensor([length, length // 2, 0], dtype=torch.int32)
    tokens = torch.randn(3, length + 4, width, generator=g).to(BF16)
    in4, out4 = (ops.quantize4(w.to(DEV), 64) for w in (w_in, w_out))
    wide_in, wide_out = (w.dequantize(torch.float64).cpu() for w in (in4, out4))

    x = tokens.double()
    normed = x * (x.square().mean(-1, keepdim=True) + ops.NORM_EPS).rsqrt() * norm.double()
    value, decay, gate = (normed @ wide_in.t()).split(width, -1)
    h, _ = og.scan(value, decay, gate, rate, lengths=lengths + 4)
    want = x + h @ wide_out.t()

    dev = tokens.to(DEV)
    with torch.inference_mode():
        normed, _ = ops.rms_norm(dev[:, :length].contiguous(), norm.to(DEV))
        proj = normed @ in4.dequantize(BF16).t()
        parts = proj.split(width, -1)
        y, state = ops.gated_scan(*parts, rate.to(DEV), lengths=lengths.to(DEV))
        prefill = dev[:, :length] + y @ out4.dequantize(BF16).t()
        rows, steps = torch.arange(3, device=DEV), []
        for i in range(4):
            row = dev[rows, lengths.to(DEV).long() + i]
            value, decay, gate = ops.linear4(row, in4, norm_weight=norm.to(DEV)).split(width, -1)
            y, state = ops.gated_step(value, decay, state, gate, rate.to(DEV), inplace=True)
            steps.append(ops.linear4(y, out4, row))
    scale = want.abs().max().item()
    for b, n in enumerate(lengths.tolist()):
        got = torch.cat([prefill[b, :n], torch.stack([s[b] for s in steps])]).double().cpu()
        assert (got - want[b, :n + 4]).abs().max().item() <= 4 * 2.0 ** -8 * 2 * scale


def _normed(x, nw, eps=1e-5):
    """RMSNorm rows in 64 bits, the norm's weight as the operator takes it (in x's dtype)."""
    xd = x.double()
    return xd * nw.to(x.dtype).double() * (xd.square().mean(-1, keepdim=True) + eps).rsqrt()


@pytest.mark.parametrize("m,n,k,group", [(1, 64, 256, 128), (8, 100, 512, 64), (9, 8672, 256, 32),
                                         (16, 6200, 384, 128), (20, 520, 256, 32), (40, 6200, 256, 64),
                                         (64, 16400, 256, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_the_norm_loses_no_bits(m, n, k, group, dtype):
    """Rows with one value each: the sum has one term, so what the norm rounds stands alone. The result
    is as near to the 64-bit one as its own rounding to 16 bits, but for FP32 errors B: of the sums
    62 scale |x| times 2^-24 in each of at most 8 steps, of the factor and the product 40 * 2^-24,
    and in f16 the term's 16 held bits, 2^-17. They count twice: with v within B of w, |round(v) - w|
    <= |round(v) - v| + B <= |round(w) - v| + B <= |round(w) - w| + 2 B."""
    g = torch.Generator().manual_seed(m + n)
    packed, scales, z, wide = _weight(n, k, group, BF16, True, g)
    at = torch.randint(0, k, (m,), generator=g)
    x = torch.zeros(m, k)
    x[torch.arange(m), at] = torch.randn(m, generator=g)
    x, nw = x.to(dtype), 1 + 0.1 * torch.randn(k, generator=g)
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV))
    with torch.inference_mode():
        got = ops.linear4(x.to(DEV), weight, norm_weight=nw.to(DEV)).double().cpu()
    xd = _normed(x, nw)
    want = xd @ wide.t()
    full = scales.double().repeat_interleave(group, 1)
    bound = 8 * 62 * 2.0 ** -24 * (xd.abs() @ full.t()) + want.abs() * (
        40 * 2.0 ** -24 + (2.0 ** -17 if dtype == F16 else 0))
    assert ((got - want).abs() <= (want.to(dtype).double() - want).abs() + 2 * bound).all()


@pytest.mark.parametrize("m,n,k", [(1, 8672, 2048), (12, 2048, 1024), (64, 8672, 1024)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_normed_projection_is_off_by_its_output_s_rounding(m, n, k, dtype):
    """Over a whole projection the error's root mean square is that of rounding the 64-bit result. The
    FP32 sums add, independently, 31 / 4.6 * 2^-24 sqrt(128) = 5e-6 of the result, against a rounding of
    about 2e-4 (f16): 0.1%. Rounding the normed row to 16 bits as well would add 40%."""
    g = torch.Generator().manual_seed(k)
    packed, scales, z, wide = _weight(n, k, 128, dtype, False, g)
    x, nw = torch.randn(m, k, generator=g).to(dtype), 1 + 0.1 * torch.randn(k, generator=g)
    with torch.inference_mode():
        got = ops.linear4(x.to(DEV), ops.Weight4(packed.to(DEV), scales.to(DEV)),
                          norm_weight=nw.to(DEV)).double().cpu()
    want = _normed(x, nw) @ wide.t()
    rounding = (want.to(dtype).double() - want).square().mean().sqrt()
    assert (got - want).square().mean().sqrt() <= 1.02 * rounding


@pytest.mark.parametrize("m,n", [(1, 70), (10, 70), (40, 6200)])
@pytest.mark.parametrize("size,weight_size", [(2e4, 15.0), (6e4, 6e4), (1e-3, 1e-3), (6e-8, 1.0)])
def test_the_norm_in_f16_beyond_f16_s_products(m, n, size, weight_size):
    """x times the norm's weight outside f16's range, in rows whose norm is inside it: as
    F.rms_norm has them. Up to 2^-17 of a term (16 held bits) and FP32 errors, as in `_check`."""
    k = 384
    g = torch.Generator().manual_seed(m)
    packed, scales, z, wide = _weight(n, k, 128, F16, True, g)
    x = (size * torch.randn(m, k, generator=g).clamp(-1, 1)).to(F16)
    nw = (weight_size * (0.5 + 0.5 * torch.rand(k, generator=g))).to(F16)
    scales = (scales.double() / weight_size).clamp(2.0 ** -14).to(F16) if weight_size > 1 else scales
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1).double().view(n, -1, 128)
    wide = ((codes - z.double().unsqueeze(-1)) * scales.double().unsqueeze(-1)).flatten(1)
    with torch.inference_mode():
        got = ops.linear4(x.to(DEV), ops.Weight4(packed.to(DEV), scales.to(DEV), z.to(DEV)),
                          norm_weight=nw.to(DEV)).double().cpu()
    xd = _normed(x, nw)
    want = xd @ wide.t()
    full = scales.double().repeat_interleave(128, 1)
    bound = (128 + 3 + 41) * 2.0 ** -24 * 63 * (xd.abs() @ full.t()) + 2.0 ** -16 * (xd.abs() @ wide.abs().t())
    limit = bound + HALF[F16] * (want.abs() + bound) + 2.0 ** -25
    big = want.abs() + limit >= 65504
    assert torch.isfinite(got[~big]).all() and (~big).sum() > big.sum()
    assert ((got - want).abs() <= limit)[~big].all()


@pytest.mark.parametrize("m,n,k,group,norm", [
    # up to 16 rows: 1, 2 and 4 tile rows a wave, 4 waves; with the norm also 9 to 16 rows
    (1, 8672, 384, 32, False), (1, 8672, 384, 64, False), (16, 8672, 384, 128, False),
    (1, 8672, 384, 32, True), (1, 8672, 384, 64, True), (8, 8672, 640, 128, True),
    (9, 8672, 384, 64, True), (16, 8672, 640, 32, True),
    (1, 16400, 384, 32, False), (3, 16400, 640, 64, False), (16, 16400, 384, 128, False),
    (7, 16400, 384, 64, True), (16, 16400, 384, 128, True), (16, 16400, 384, 32, True),
    (12, 100, 384, 64, True),
    # more rows, x staged once: one team of waves, two, one and two tile rows a wave
    (256, 8672, 384, 128, False), (130, 12304, 384, 64, False), (250, 8672, 384, 32, False),
    (256, 8672, 384, 64, True), (40, 8672, 384, 128, True), (33, 28700, 256, 32, True),
    (17, 6144, 384, 128, False), (17, 6144, 384, 128, True), (200, 4000, 384, 32, True)])
@pytest.mark.parametrize("dtype,scale_dtype", [(BF16, BF16), (F16, F16), (BF16, F16), (F16, BF16)])
def test_every_form_of_the_kernels(m, n, k, group, norm, dtype, scale_dtype):
    g = torch.Generator().manual_seed(m + n + group)
    zeros = (m + n) % 2 == 0 if dtype == BF16 else (m + n) % 2 == 1
    packed, scales, z, wide = _weight(n, k, group, scale_dtype, zeros, g)
    x = torch.randn(m, k, generator=g).to(dtype)
    res = torch.randn(m, n, generator=g).to(dtype)
    nw = 1 + 0.1 * torch.randn(k, generator=g) if norm else None
    weight = ops.Weight4(packed.to(DEV), scales.to(DEV), None if z is None else z.to(DEV))
    bad = x.to(DEV).clone()
    bad[m // 2] = float("nan")
    dev = None if nw is None else nw.to(DEV)
    with torch.inference_mode():
        got = ops.linear4(x.to(DEV), weight, res.to(DEV), norm_weight=dev)
        _check(got, x, wide, scales, group, res, nw)
        spoilt = ops.linear4(bad, weight, res.to(DEV), norm_weight=dev)
    keep = [i for i in range(m) if i != m // 2]
    assert torch.equal(got[keep], spoilt[keep]) and torch.isnan(spoilt[m // 2]).all()


def test_a_step_in_another_type_than_the_weights_is_refused():
    """As without 4-bit copies: rows of the other 16-bit type do not run on them."""
    model = Mamba3(256, d_state=128, depth=1).eval().to(DEV, F16)
    x = torch.zeros(1, 1, 256, device=DEV, dtype=BF16)
    with torch.inference_mode():
        for _ in range(2):
            with pytest.raises(RuntimeError):
                model.step(x, None)
            model.quantize_decode()
