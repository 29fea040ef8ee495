"""``m3_rows8`` (``ops.quantize8_rows``, ``ops.rms_norm8``) against quotients and norms in 64 bits.

Codes are exact: the nearest integers of 127 p / max|p|, ties to even, told by quotient and remainder in
64 bits (p = s * w has 48 bits at most, 127 p 55 of which FP64 keeps 53: such a tie of FP32 rows is
made on purpose only where it is exact). Scales are off by the quotient's and the product's half steps, 2 *
2^-24, and with the norm by the factor's: half the error of a sum of squares of positive terms, each of which
passes at most dim / 64 + 24 additions, and 4 steps of the mean, eps and reciprocal root.
"""

from __future__ import annotations

import pytest
import torch

from mamba3_amd import _hip, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


def _codes(p):
    """p [M, K] in 64 bits -> exact codes, and max|p|."""
    most = p.abs().amax(1, keepdim=True)
    part = 127 * p.abs()
    safe = torch.where(most > 0, most, 1.0)
    whole = torch.floor(part / safe)
    twice = 2 * (part - whole * safe)
    up = (twice > safe) | ((twice == safe) & (whole % 2 == 1))
    return torch.where(most > 0, torch.sign(p) * (whole + up), 0.0), most.squeeze(1)


def _want(x, weight=None, add=None, eps=EPS):
    s = x if add is None else (x.float() + add.float()).to(x.dtype)
    if weight is None:
        codes, most = _codes(s.double())
        return codes, most / 127, s
    codes, most = _codes(s.double() * weight.to(x.dtype).double())
    return codes, most / 127 * (s.double().square().mean(1) + eps).rsqrt(), s


def _check(got, x, weight=None, add=None, eps=EPS):
    rows, total = got
    codes, scales, s = _want(x, weight, add, eps)
    k = x.shape[-1]
    assert torch.equal(rows.codes.cpu().double(), codes)
    bound = 2 + (0 if weight is None else (k / 64 + 24) / 2 + 4)
    # below FP32's normal range half its smallest step
    assert ((rows.scales.cpu().double() - scales).abs() <= bound * 2.0 ** -24 * scales + 2.0 ** -149).all()
    if total is not None:
        assert torch.equal(total.cpu(), s)


DIMS = [1, 2, 7, 8, 9, 64, 65, 120, 128, 129, 250, 256, 257, 511, 512, 513, 1000, 1024, 1111, 2048, 2049, 4096, 5003, 8192, 8199, 16400]


def _inputs(m, k, dtype, g):
    x = torch.randn(m, k, generator=g)
    x[:, ::5] *= 0.01
    return x.to(dtype)


@pytest.mark.parametrize("k", DIMS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows(k, dtype):
    g = torch.Generator().manual_seed(k)
    for m in (1, 5, 37):
        x = _inputs(m, k, dtype, g)
        with torch.inference_mode():
            _check((ops.quantize8_rows(x.to(DEV)), None), x)


@pytest.mark.parametrize("k", DIMS)
@pytest.mark.parametrize("dtype,add_dtype", [(F32, None), (F32, F32), (F32, BF16), (F32, F16), (BF16, None),
                                             (BF16, BF16), (F16, None), (F16, F16)])
def test_normed_rows(k, dtype, add_dtype):
    g = torch.Generator().manual_seed(k + 1)
    weight = (1 + 0.2 * torch.randn(k, generator=g)).to([F32, BF16, F16][k % 3])
    for m in (1, 38):
        x = _inputs(m, k, dtype, g)
        add = None if add_dtype is None else torch.randn(m, k, generator=g).to(add_dtype)
        dev = [None if t is None else t.to(DEV) for t in (x, weight, add)]
        for keep in (False, True) if add is not None else (False,):
            with torch.inference_mode():
                got = ops.rms_norm8(dev[0], dev[1], EPS, add=dev[2], keep_sum=keep)
            assert (got[1] is not None) == keep
            _check(got, x, weight, add)


@pytest.mark.parametrize("m,k,dtype", [(3000, 1024, BF16), (1029, 2048, F16), (515, 4096, F32), (3, 131071, F32),
                                       (2, 131071, BF16)])
def test_many_rows(m, k, dtype):
    """Enough elements that some lie within 1e-4 of half a code: these are settled apart."""
    g = torch.Generator().manual_seed(m)
    x = _inputs(m, k, dtype, g)
    weight, add = 1 + 0.2 * torch.randn(k, generator=g), torch.randn(m, k, generator=g).to(dtype)
    p = x.double() * 127 / x.double().abs().amax(1, keepdim=True)
    assert ((p - p.floor() - 0.5).abs() < 1e-4).any()
    with torch.inference_mode():
        _check((ops.quantize8_rows(x.to(DEV)), None), x)
        _check(ops.rms_norm8(x.to(DEV), weight.to(DEV), EPS, add=add.to(DEV), keep_sum=True), x, weight, add)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("norm", [False, True])
def test_halves_go_to_even(dtype, norm):
    """Rows whose greatest value is 127 times a power of two: their codes' halves are values of each type."""
    halves = torch.arange(-126.5, 127, 1.0)
    rows = torch.stack([torch.cat([halves, torch.tensor([s * 127.0])]) * 2.0 ** e for s, e in
                        ((1, 0), (-1, 3), (1, -9), (-1, -5))]).to(dtype)
    weight = torch.ones(rows.shape[1]) * 0.25
    with torch.inference_mode():
        got = (ops.rms_norm8(rows.to(DEV), weight.to(DEV))[0] if norm
               else ops.quantize8_rows(rows.to(DEV)))
    want = torch.cat([halves, torch.tensor([127.0])]).round().repeat(4, 1)  # torch rounds halves to even
    want[1, -1] = want[3, -1] = -127
    assert torch.equal(got.codes.cpu().float(), want)


@pytest.mark.parametrize("norm", [False, True])
def test_beside_a_half(norm):
    """FP32 values next to half a code on either side, where 127 x / max|x| in FP32 cannot tell."""
    g = torch.Generator().manual_seed(5)
    most = 1 + torch.rand(64, 1, generator=g)
    weight = 1 + torch.rand(256, generator=g) if norm else torch.ones(256)
    code = torch.randint(0, 127, (64, 256), generator=g).float() + 0.5
    x = (code.double() * most.double() / 127 / weight.double()).float()
    steps = torch.randint(-2, 3, (64, 256), generator=g)
    x = (x.view(torch.int32) + steps.int()).view(F32)
    x[:, 7] = most[:, 0] / weight[7] * 1.0001
    if norm:
        with torch.inference_mode():
            _check(ops.rms_norm8(x.to(DEV), weight.to(DEV)), x, weight)
    else:
        with torch.inference_mode():
            _check((ops.quantize8_rows(x.to(DEV)), None), x)


@pytest.mark.parametrize("k", [40, 600, 3000, 9001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_zeros_infinities_and_nan(k, dtype):
    g = torch.Generator().manual_seed(k)
    x = _inputs(7, k, dtype, g)
    x[0], x[2, 3], x[3, k - 1], x[4, 5], x[5, 0] = 0, float("inf"), float("nan"), -float("inf"), float("nan")
    weight = torch.ones(k)
    with torch.inference_mode():
        for rows in (ops.quantize8_rows(x.to(DEV)), ops.rms_norm8(x.to(DEV), weight.to(DEV))[0]):
            codes, scales = rows.codes.cpu(), rows.scales.cpu()
            assert not codes[[0, 2, 3, 4, 5]].any()
            assert scales[0] == 0 and torch.isnan(scales[2:6]).all()
            good = x[[1, 6]]
            assert torch.equal(codes[[1, 6]].double(), _codes(good.double())[0])
        weight[k // 2] = float("nan")
        rows = ops.rms_norm8(x.to(DEV), weight.to(DEV))[0]
        assert torch.isnan(rows.scales[[1, 6]]).all() and not rows.codes.any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_small_and_great_rows(dtype):
    """Rows at both ends of the type's range, subnormal ones among them."""
    g = torch.Generator().manual_seed(9)
    info = torch.finfo(dtype)
    x = torch.rand(6, 200, generator=g).double() + 0.1
    for i, most in enumerate((info.max, info.max / 3, info.tiny, info.tiny * 4, info.smallest_normal * info.eps * 40,
                              1e-30 if dtype != F16 else 1e-4)):
        x[i] *= most / x[i].max()
    x = x.to(dtype)
    with torch.inference_mode():
        _check((ops.quantize8_rows(x.to(DEV)), None), x)


def test_strides_and_shapes():
    """Slices at odd offsets, rows apart, more axes, a column of a transposed tensor; the neighbours
    of what is read stay out of it."""
    g = torch.Generator().manual_seed(2)
    base = torch.full((4, 9, 301), float("nan"))
    base[:, :, 7:207] = torch.randn(4, 9, 200, generator=g)
    weight = torch.full((250,), float("nan"))
    weight[3:203] = 1 + 0.1 * torch.randn(200, generator=g)
    for dtype in (F32, BF16, F16):
        x = base.to(dtype)[:, :, 7:207]
        dev = base.to(DEV, dtype)[:, :, 7:207]
        w = weight.to(DEV)[3:203]
        with torch.inference_mode():
            rows, total = ops.rms_norm8(dev, w, add=dev, keep_sum=True)
            assert rows.shape == (4, 9, 200) == rows.codes.shape and rows.scales.shape == (4, 9)
            flat = x.reshape(36, 200)
            _check((ops.Rows8(rows.codes.flatten(0, 1), rows.scales.flatten()), total.flatten(0, 1)),
                   flat, weight[3:203], flat)
            turned = ops.quantize8_rows(dev.transpose(0, 2))
            assert torch.equal(turned.codes.cpu().double().flatten(0, 1),
                               _codes(x.transpose(0, 2).reshape(-1, 4).double())[0])
            one = ops.quantize8_rows(dev[1, 2])
            assert one.shape == (200,) and one.scales.shape == ()
            assert torch.equal(one.codes.cpu().double(), _codes(flat[11:12].double())[0][0])
            assert torch.equal(one.dequantize(F16),
                               (one.codes.float() * one.scales).to(F16))
            none = ops.rms_norm8(dev[:0], w, add=dev[:0], keep_sum=True)
            assert none[0].shape == (0, 9, 200) and none[1].shape == (0, 9, 200)


@pytest.mark.parametrize("k", [1, 3, 4, 5, 8, 31, 100, 1024, 1111, 2049, 8200])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, torch.float64])
def test_values(k, dtype):
    """What the rows stand for, the same FP32 product and rounding as torch's; a NaN scale's row is NaN."""
    g = torch.Generator().manual_seed(k)
    for m in (1, 7, 300):
        codes = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
        scales = torch.rand(m, generator=g) / 100
        scales[m // 2] = float("nan")
        got = ops.Rows8(codes.to(DEV), scales.to(DEV)).dequantize(dtype)
        want = (codes.float() * scales.unsqueeze(1)).to(dtype)
        assert got.dtype == dtype and torch.equal(got.cpu().nan_to_num(9.0), want.nan_to_num(9.0))
        assert torch.isnan(got[m // 2]).all()


@pytest.mark.parametrize("k", [1, 100, 2048, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_zeros_without_eps(k, dtype):
    """eps = 0: a row of zeros is NaN, as F.rms_norm's; the next row and any eps above 0 know nothing of it."""
    x = torch.zeros(3, k, dtype=dtype, device=DEV)
    x[1] = 0.5
    weight = torch.ones(k, device=DEV)
    rows, _ = ops.rms_norm8(x, weight, 0.0)
    assert torch.isnan(rows.scales[::2]).all() and (rows.codes[::2] == 0).all()
    assert torch.isnan(torch.nn.functional.rms_norm(x, (k,), weight.to(dtype), 0.0)[::2]).all()
    # 0.5 / 127 / 0.5: a rounding of 127ths, one of the root (2 steps), one of the product
    assert (rows.codes[1] == 127).all() and abs(rows.scales[1].item() * 127 - 1) < 5 * 2 ** -24
    rows, _ = ops.rms_norm8(x, weight, EPS)
    assert (rows.scales[::2] == 0).all() and (rows.codes[::2] == 0).all()


def test_what_is_written():
    """The C entry point: codes and scales of the rows and nothing else; the sum in x's place, or the add's."""
    g = torch.Generator().manual_seed(3)
    for k in (77, 2500, 9000):
        whole = -(-k // 16) * 16
        x = torch.randn(5, k, generator=g).to(BF16)
        add = torch.randn(5, k, generator=g).to(BF16)
        weight = torch.ones(k)
        for place in ("x", "add", "own"):
            dev = dict(x=x.to(DEV), add=add.to(DEV), own=torch.zeros(5, k, dtype=BF16, device=DEV))
            codes = torch.full((7, whole + 32), 99, dtype=torch.int8, device=DEV)
            scales = torch.full((7,), 99.0, device=DEV)
            w = weight.to(DEV)
            args = _hip.Rows8Args(5, k, EPS, 0, _hip.tensor(dev["x"]), _hip.tensor(dev["add"]),
                                  _hip.tensor(w), _hip.tensor(dev[place]), codes.data_ptr(), whole + 32,
                                  scales.data_ptr())
            _hip.call("m3_rows8", args, DEV)
            want, _, s = _want(x, weight, add)
            assert torch.equal(codes[:5, :k].cpu().double(), want)
            assert (codes[5:] == 99).all() and (codes[:, whole:] == 99).all() and (scales[5:] == 99).all()
            assert torch.equal(dev[place].cpu(), s)
            for name, given in (("x", x), ("add", add)):
                assert name == place or torch.equal(dev[name].cpu(), given)


def test_gradients_are_refused_not_dropped():
    x = torch.randn(4, 40, device=DEV, requires_grad=True)
    weight = torch.ones(40, device=DEV)
    for call in (lambda: ops.quantize8_rows(x), lambda: ops.rms_norm8(weight.expand(4, 40), weight, add=x),
                 lambda: ops.rms_norm8(x.detach(), x[0]),
                 lambda: ops.linear8(ops.quantize8_rows(x.detach()), ops.quantize8(x.detach()), x[:, :4],
                                     dtype=F32),
                 lambda: ops.linear8(ops.Rows8(torch.zeros(4, 40, dtype=torch.int8, device=DEV), x[:, 0]),
                                     ops.quantize8(x.detach()))):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with torch.no_grad():
        ops.rms_norm8(x, weight, add=x, keep_sum=True)


def test_rows_that_are_one_row():
    """Expanded inputs: rows with a stride of 0."""
    g = torch.Generator().manual_seed(11)
    x, add = torch.randn(1, 300, generator=g).to(F16), torch.randn(1, 300, generator=g).to(F16)
    weight = torch.tensor([0.5])
    with torch.inference_mode():
        got = ops.rms_norm8(x.to(DEV).expand(9, 300), weight.to(DEV).expand(300), add=add.to(DEV).expand(9, 300),
                            keep_sum=True)
        _check(got, x.expand(9, 300), weight.expand(300), add.expand(9, 300))


def test_more_rows_than_a_launch_has_threads():
    """2^28 rows of 16 lanes each, and what they stand for by one lane each: the last rows are the last."""
    rows = (1 << 28) + 37
    x = torch.ones(rows, 2, dtype=BF16, device=DEV)
    x[:, 1] = 0.25
    x[-5:] = torch.tensor([[1.0, -3.0]], dtype=BF16)
    with torch.inference_mode():
        got = ops.quantize8_rows(x)
        assert (got.codes[:1000] == torch.tensor([127, 32], device=DEV)).all()
        assert (got.codes[-1000:-5] == torch.tensor([127, 32], device=DEV)).all()
        assert (got.codes[-5:] == torch.tensor([42, -127], device=DEV)).all()
        tail = ops.Rows8(got.codes, got.scales).dequantize(BF16)[-6:].float()
    want = torch.tensor([[1.0, 32 / 127]] + [[42 * 3 / 127, -3.0]] * 5)
    assert ((tail.cpu() - want).abs() <= 2.0 ** -8 * want.abs()).all()


def test_streams_and_graphs():
    """On a stream of its own, and captured and replayed with new inputs between eager calls."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(33, 1000, generator=g).to(BF16)
    weight = torch.ones(1000, device=DEV)
    static = torch.zeros(33, 1000, dtype=BF16, device=DEV)
    side = torch.cuda.Stream()
    with torch.inference_mode():
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            rows = ops.quantize8_rows(x.to(DEV))
        side.synchronize()
        _check((rows, None), x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = ops.rms_norm8(static, weight, add=static, keep_sum=True)
        for i in range(3):
            new = torch.randn(33, 1000, generator=g).to(BF16)
            static.copy_(new)
            graph.replay()
            eager = ops.rms_norm8(static, weight, add=static, keep_sum=True)
            torch.cuda.synchronize()
            _check(held, new, weight.cpu(), new)
            assert torch.equal(eager[0].codes, held[0].codes) and torch.equal(eager[0].scales, held[0].scales)
