"""``m3_linear8`` (``ops.linear8``, ``ops.Weight8``) against the product in 64 bits.

Sums of codes are exact integers below 2^31. A result then has, in FP32, the sum's rounding, two products' and
(with a residual) an addition's, 2^-24 each, and half a step of its own type.
"""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import Mamba3, _hip, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _operands(m, n, k, g, full=False):
    low = -128 if full else -127
    codes = torch.randint(low, 128, (m, k), generator=g, dtype=torch.int8)
    q = torch.randint(low, 128, (n, k), generator=g, dtype=torch.int8)
    rs = (0.5 + torch.rand(m, generator=g)) / 64
    s = (0.5 + torch.rand(n, generator=g)) / (64 * k ** 0.5)
    return codes, q, rs, s


def _check(got, codes, q, rs, s, residual=None):
    """On the GPU, where FP64 holds the sums exactly."""
    codes, q, rs, s = (t.to(DEV).double() for t in (codes, q, rs, s))
    product = codes @ q.t().contiguous() * rs.unsqueeze(1) * s
    want = product if residual is None else product + residual.to(DEV).double()
    slack = 3 * 2.0 ** -24 * product.abs() + 2.0 ** -24 * want.abs()
    limit = slack + HALF[got.dtype] * (want.abs() + slack) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    worst = ((got.double() - want).abs() / limit).max().item()
    assert worst <= 1.0, f"error / bound = {worst:.3f}"


SHAPES = [(1, 1, 1), (1, 17, 15), (2, 64, 16), (3, 65, 17), (5, 1111, 1120), (7, 130, 63), (15, 63, 64),
          (16, 2048, 1024), (17, 33, 65), (31, 48, 2048), (33, 260, 127), (48, 130, 128), (64, 512, 4096),
          (65, 40, 129), (100, 257, 300), (129, 129, 1111), (130, 640, 256), (256, 31, 640), (257, 300, 191),
          (511, 1000, 96), (777, 65, 33)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear8(shape, dtype, residual):
    m, n, k = shape
    g = torch.Generator().manual_seed(m + 7 * n + k)
    codes, q, rs, s = _operands(m, n, k, g, full=True)
    res = torch.randn(m, n, generator=g).to(dtype) if residual else None
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(codes.to(DEV), rs.to(DEV)), weight,
                          None if res is None else res.to(DEV), dtype=dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    _check(got, codes, q, rs, s, res)


@pytest.mark.parametrize("m,n,k,dtype", [
    (1, 28672, 8192, BF16), (4, 8672, 2048, F16), (256, 8672, 2048, BF16), (64, 64, 65536, F32),
    (300, 28672, 640, BF16), (5000, 4480, 1024, BF16), (4096, 4097, 250, F16), (2049, 16385, 128, F32),
    (70000, 192, 64, BF16), (33000, 1, 40, F32)])
def test_large(m, n, k, dtype):
    g = torch.Generator().manual_seed(k)
    codes, q, rs, s = _operands(m, n, k, g)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(codes.to(DEV), rs.to(DEV)), weight, dtype=dtype)
    step = max(1, (1 << 26) // n)
    for at in range(0, m, step):
        _check(got[at:at + step], codes[at:at + step], q, rs[at:at + step], s)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_the_longest_sums(m):
    """K = 131071 products of -128 and -128: 2^31 - 16384, the greatest sum there is, exactly."""
    k = _hip.LINEAR8_MAX_K
    codes = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    weight = ops.Weight8(torch.full((70, k), -128, dtype=torch.int8, device=DEV), torch.ones(70, device=DEV))
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(codes, torch.ones(m, device=DEV)), weight, dtype=F32)
    assert (got == float(k * 16384)).all()


@pytest.mark.parametrize("m", [3, 20, 70, 300])
def test_one_column_at_a_time(m):
    """Rows with a single code read one column: every code of the weight comes back in its place."""
    g = torch.Generator().manual_seed(m)
    q = torch.randint(-127, 128, (150, 200), generator=g, dtype=torch.int8).to(DEV)
    weight = ops.Weight8(q, torch.ones(150, device=DEV))
    at = torch.randint(0, 200, (m,), generator=g).to(DEV)
    codes = torch.zeros(m, 200, dtype=torch.int8, device=DEV)
    codes[torch.arange(m, device=DEV), at] = 1
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(codes, torch.ones(m, device=DEV)), weight, dtype=F32)
    assert torch.equal(got, q.t()[at].float())


@pytest.mark.parametrize("m", [2, 50, 70, 600])
def test_rows_that_are_not_numbers(m):
    """A row whose scale is NaN is NaN, and no other; what lies behind a row's codes has no effect."""
    g = torch.Generator().manual_seed(m)
    codes, q, rs, s = _operands(m, 100, 90, g)
    wide = torch.full((m, 128), 55, dtype=torch.int8, device=DEV)
    wide[:, :90] = codes.to(DEV)
    bad = rs.clone()
    bad[m // 2] = float("nan")
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(wide[:, :90], bad.to(DEV)), weight)
    assert torch.isnan(got[m // 2]).all()
    keep = [i for i in range(m) if i != m // 2]
    _check(got[keep], codes[keep], q, rs[keep], s)


@pytest.mark.parametrize("m", [9, 60, 200, 700])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_strided_operands(m, dtype):
    """Codes, residual and out in rows apart and at odd offsets; out as the residual; rows behind
    the last and columns beside them as they were."""
    g = torch.Generator().manual_seed(m)
    n, k = 203, 140
    codes, q, rs, s = _operands(m, n, k, g)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    base = torch.full((m, k + 37), 77, dtype=torch.int8, device=DEV)
    base[:, 5:5 + k] = codes.to(DEV)
    out = torch.full((m + 3, n + 13), 7.0, dtype=dtype, device=DEV)
    res = torch.randn(m, n, generator=g).to(dtype)
    base_res = torch.zeros(m, n + 9, dtype=dtype, device=DEV)
    base_res[:, 3:3 + n] = res.to(DEV)
    rows = ops.Rows8(base[:, 5:5 + k], rs.to(DEV))
    with torch.inference_mode():
        back = ops.linear8(rows, weight, base_res[:, 3:3 + n], out=out[:m, 5:5 + n])
        assert back.data_ptr() == out[:m, 5:5 + n].data_ptr()
        _check(out[:m, 5:5 + n], codes, q, rs, s, res)
        assert (out[m:] == 7).all() and (out[:, :5] == 7).all() and (out[:, 5 + n:] == 7).all()
        ops.linear8(rows, weight, base_res[:, 3:3 + n], out=base_res[:, 3:3 + n])
        assert torch.equal(base_res[:, 3:3 + n], out[:m, 5:5 + n])


@pytest.mark.parametrize("k", [1, 3, 15, 16, 17, 40, 63, 100, 129, 200, 333, 1111])
@pytest.mark.parametrize("m,n", [(1, 70), (3, 9000), (15, 64), (16, 130), (17, 1), (33, 9000), (100, 500), (260, 1500),
                                 (700, 5000), (3000, 2500)])
def test_codes_at_any_alignment(m, n, k):
    """Rows side by side of any width, at an odd address, that end where their memory does; and apart."""
    g = torch.Generator().manual_seed(m + k)
    codes, q, rs, s = _operands(m, n, k, g, full=True)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    odd = torch.empty(m * k + 5, dtype=torch.int8, device=DEV)[5:].view(m, k)
    odd.copy_(codes)
    apart = torch.full((m, k + 7), 3, dtype=torch.int8, device=DEV)[:, 7:]
    apart.copy_(codes)
    with torch.inference_mode():
        first = ops.linear8(ops.Rows8(odd, rs.to(DEV)), weight)
        _check(first, codes, q, rs, s)
        for given in (apart, codes.to(DEV)):
            assert torch.equal(ops.linear8(ops.Rows8(given, rs.to(DEV)), weight), first)


@pytest.mark.parametrize("m,n,k", [(13000, 1, 17), (20000, 63, 90), (20011, 64, 333), (13000, 65, 90), (2097120, 3, 17),
                                   (2097121, 3, 17)])
def test_many_rows_at_any_alignment(m, n, k):
    """Few outputs of many rows, on both sides of 64 columns and of 65,535 rows of workgroups; with a residual."""
    g = torch.Generator().manual_seed(m + k)
    codes, q, rs, s = _operands(m, n, k, g)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    res = torch.randn(m, n, generator=g).to(F16)
    odd = torch.empty(m * k + 3, dtype=torch.int8, device=DEV)[3:].view(m, k)
    odd.copy_(codes)
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(odd, rs.to(DEV)), weight, res.to(DEV))
        _check(got, codes, q, rs, s, res)
        assert torch.equal(ops.linear8(ops.Rows8(codes.to(DEV), rs.to(DEV)), weight, res.to(DEV)), got)


def test_more_axes_and_no_rows():
    g = torch.Generator().manual_seed(6)
    codes, q, rs, s = _operands(6, 40, 50, g)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    flat = ops.linear8(ops.Rows8(codes.to(DEV), rs.to(DEV)), weight)
    cube = ops.linear8(ops.Rows8(codes.view(2, 3, 50).to(DEV), rs.view(2, 3).to(DEV)), weight)
    one = ops.linear8(ops.Rows8(codes[4].to(DEV), rs[4].to(DEV)), weight)
    none = ops.linear8(ops.Rows8(codes[:0].to(DEV), rs[:0].to(DEV)), weight)
    assert cube.shape == (2, 3, 40) and one.shape == (40,) and none.shape == (0, 40)
    assert torch.equal(cube.view(6, 40), flat) and torch.equal(one, flat[4]) and flat.dtype == BF16


def test_offsets_past_32_bits():
    """Codes and outputs of over 2^31 bytes and elements: the last rows are the last rows."""
    m, n, k = 70000, 32800, 32832
    codes = torch.zeros(m, k, dtype=torch.int8, device=DEV)
    codes[-3:, 100:110] = 3
    q = torch.ones(n, k, dtype=torch.int8, device=DEV)
    weight = ops.Weight8(q, torch.ones(n, device=DEV))
    rs = torch.ones(m, device=DEV)
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(codes, rs), weight)
    assert got.numel() > 1 << 31 and (got[-3:] == 30).all() and not got[-2000:-3].any() and not got[:2000].any()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [5000, 5003])
def test_every_kernel_gives_the_same_bits(n, dtype, residual):
    """Sums are exact, and an output's operations the same in all kernels: a row's result does not depend
    on how many rows come with it."""
    g = torch.Generator().manual_seed(8)
    codes, q, rs, s = _operands(3000, n, 333, g)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    res = torch.randn(3000, n, generator=g).to(dtype).to(DEV) if residual else None
    with torch.inference_mode():
        whole = ops.linear8(ops.Rows8(codes.to(DEV), rs.to(DEV)), weight, res, dtype=dtype)
        _check(whole, codes, q, rs, s, res)
        for m in (1, 2, 16, 17, 40, 64, 65, 128, 200, 500, 700, 1500):
            part = ops.linear8(ops.Rows8(codes[:m].to(DEV), rs[:m].to(DEV)), weight,
                               None if res is None else res[:m], dtype=dtype)
            assert torch.equal(part, whole[:m]), m


def _product(codes, scales, weight):
    """Rows and a Weight8 in 64 bits, summed in whole codes: sums of rounded code * scale leave something
    where the codes' sum is 0. A code of the weight is the integer nearest to its rounded value / scale."""
    w_scales = weight.scales[:weight.shape[0]]
    q = (weight.dequantize() / w_scales.unsqueeze(1)).round().double()
    return codes.to(DEV) @ q.t().contiguous() * scales.to(DEV).unsqueeze(1) * w_scales.double()


def test_streams_and_graphs():
    g = torch.Generator().manual_seed(4)
    codes, q, rs, s = _operands(200, 300, 256, g)
    weight = ops.Weight8(q.to(DEV), s.to(DEV))
    static = torch.zeros(200, 256, dtype=torch.int8, device=DEV)
    scales = rs.to(DEV)
    side = torch.cuda.Stream()
    with torch.inference_mode():
        ops.linear8(ops.Rows8(static, scales), weight)
        side.wait_stream(torch.cuda.current_stream())
        graphs = []
        for m in (4, 200):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = ops.linear8(ops.Rows8(static[:m], scales[:m]), weight)
            graphs.append((graph, held, m))
        for i in range(3):
            new = torch.randint(-127, 128, (200, 256), generator=g, dtype=torch.int8)
            static.copy_(new)
            for graph, held, m in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for graph, held, m in graphs:
                _check(held, new[:m], q, rs[:m], s)


@pytest.mark.parametrize("m,width,inner", [(1, 200, 400), (50, 96, 130), (400, 250, 333)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_a_block_s_projections(m, width, inner, dtype):
    """The operators as a block runs them: residual add, norm and rounding, in_proj, an elementwise
    mixer, rounding, out_proj with the residual; against the same in 64 bits with the codes of each step
    (so that no code is in doubt). Each product's bound is test_linear8's; the first's scales are the
    norm's, off by up to (width / 64 + 24) / 2 + 6 steps of FP32."""
    from test_gpu_rows8 import _want
    g = torch.Generator().manual_seed(width)
    x, add = (torch.randn(m, width, generator=g).to(dtype) for _ in range(2))
    norm = 1 + 0.1 * torch.randn(width, generator=g)
    in8 = ops.quantize8((torch.randn(inner, width, generator=g) / width ** 0.5).to(DEV))
    out8 = ops.quantize8((torch.randn(width, inner, generator=g) / inner ** 0.5).to(DEV))
    with torch.inference_mode():
        rows, stream = ops.rms_norm8(x.to(DEV), norm.to(DEV), add=add.to(DEV), keep_sum=True)
        proj = ops.linear8(rows, in8, dtype=dtype)
        mixed = torch.nn.functional.silu(proj)
        again = ops.quantize8_rows(mixed)
        y = ops.linear8(again, out8, stream, dtype=dtype)
    codes, scales, s = _want(x, norm, add)
    wide = _product(codes, scales, in8)
    steps = ((width / 64 + 24) / 2 + 10) * 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == F16 else 1e-37
    assert ((proj.double() - wide).abs() <= (HALF[dtype] + steps) * (1 + steps) * wide.abs() + tiny).all()
    codes, scales, _ = _want(mixed.cpu())
    part = _product(codes, scales, out8)
    want = part + s.to(DEV).double()
    slack = 8 * 2.0 ** -24 * part.abs() + 2.0 ** -24 * want.abs()
    assert ((y.double() - want).abs() <= slack + HALF[dtype] * (want.abs() + slack) + tiny).all()


def _layer8(model, h, mixed, layer, dtype, cache):
    """One layer of a model whose projections are in 8 bits, by the operators."""
    rows, s = ops.rms_norm8(h, layer.norm.weight, layer.norm.eps, add=mixed, keep_sum=mixed is not None)
    mixer = layer.mixer
    in8, out8 = (ops.quantize8(getattr(mixer, name).weight) for name in ("in_proj", "out_proj"))
    proj = ops.linear8(rows, in8, dtype=dtype)
    y, state, phase, k = ops.scan_projection(proj, mixer, want_cache=True, chunk_size=mixer._chunk())
    return ops.linear8(ops.quantize8_rows(y.flatten(-2)), out8, dtype=dtype), h if mixed is None else s, state


@pytest.mark.parametrize("width,dtype,autocast", [(256, F32, BF16), (96, BF16, None), (512, F16, None),
                                                  (160, F32, None)])
def test_quantize_prefill(width, dtype, autocast):
    """forward and prefill are the operators' composition, bit for bit, and stay within the rounding of
    8 bits of the model that is not rounded: each of a layer's two projections has operands off by up to half a
    code of 127 on either side, about 2 / 254 of the greatest value of rows of some 4 standard deviations, that is
    2 * 4 / 254 / sqrt(3) = 2% of the result's size in the mean; 4 layers' sums of both at most 4 * 2 * 2%."""
    torch.manual_seed(width)
    model = Mamba3(width, d_state=64, depth=2).eval().to(DEV, dtype)
    x = torch.randn(3, 70, width, device=DEV, dtype=dtype)
    with torch.inference_mode(), torch.autocast("cuda", dtype=autocast or BF16, enabled=autocast is not None):
        plain = model(x)
        cache0 = model.prefill(x)[1]
        model.quantize_prefill()
        got, (y, cache) = model(x), model.prefill(x)
        h, mixed = x, None
        for i, layer in enumerate(model.layers):
            mixed, h, state = _layer8(model, h, mixed, layer, autocast or dtype, cache)
            assert torch.equal(state, cache[i][1])
        want = model._add_norm(h, mixed, model.norm_f, torch.promote_types(h.dtype, mixed.dtype), False)[0]
    assert torch.equal(got, y) and torch.equal(got, want) and got.dtype == plain.dtype
    assert not torch.equal(got, plain)
    assert (got.double() - plain.double()).norm() <= 4 * 2 * 0.02 * plain.double().norm()
    assert [[t.dtype for t in c] for c in cache] == [[t.dtype for t in c] for c in cache0]


def test_quantize_prefill_steps_and_graphs():
    """Steps of up to 64 rows are as they were, those of more run in 8 bits, eager and captured; the
    prefill's cache continues in either."""
    torch.manual_seed(0)
    model = Mamba3(256, d_state=64, depth=2).eval().to(DEV, BF16)
    x = torch.randn(80, 6, 256, device=DEV, dtype=BF16)
    with torch.inference_mode():
        few, _ = model.step(x[:5, :1])
        many, _ = model.step(x[:, :1])
        model.quantize_prefill()
        assert torch.equal(model.step(x[:5, :1])[0], few)
        y, cache = model.prefill(x[:, :4])
        steps = []
        for t in (4, 5):
            out, cache = model.step(x[:, t:t + 1], cache)
            steps.append(out)
        first, _ = model.step(x[:, :1])
        assert not torch.equal(first, many)
        # a step and a prefill of one token differ by roundings alone: the step kernel's, and codes beside them
        one, _ = model.prefill(x[:, :1])
        assert (first.float() - one.float()).norm() <= 0.05 * one.float().norm()
        graph = model.cuda_graph(80)
        for _ in range(2):
            graph.load_cache(model.prefill(x[:, :4])[1])
            for t, want in zip((4, 5), steps):
                assert torch.equal(graph(x[:, t:t + 1]), want)


def test_quantize_prefill_both_directions():
    torch.manual_seed(1)
    model = Mamba3(192, d_state=32, depth=2, causal=False).eval().to(DEV, F16)
    x = torch.randn(2, 90, 192, device=DEV, dtype=F16)
    with torch.inference_mode():
        plain = model(x)
        got = model.quantize_prefill()(x)
        assert torch.equal(got, model(x))
    assert not torch.equal(got, plain) and (got.float() - plain.float()).norm() <= 0.16 * plain.float().norm()


def test_a_changed_weight_is_refused():
    model = Mamba3(128, depth=1).eval().to(DEV, BF16).quantize_prefill()
    x = torch.randn(2, 5, 128, device=DEV, dtype=BF16)
    with torch.inference_mode():
        model(x)
        with pytest.raises(RuntimeError):  # rows of another type than the weights', as without copies
            model(x.half())
    with torch.no_grad():
        model.layers[0].mixer.out_proj.weight.mul_(2)
    with torch.inference_mode(), pytest.raises(RuntimeError, match="call it again"):
        model(x)
