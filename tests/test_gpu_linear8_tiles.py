"""``m3_linear8``'s kernels for many rows, each with outputs that it writes whole (16 bytes a lane) and at any alignment,
with one tile of out a workgroup and with several, against the product in 64 bits.

The bound is that of the few rows' tests: sums are exact, then three roundings to FP32 of the product, one of its
sum with a residual, and half a step of the result's own type.
"""

from __future__ import annotations

import functools

import pytest
import torch

from mamba3_amd import _hip, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
CUS = 256


def _form(m, n, k):
    """The kernel that a call of aligned rows takes, as the library's rule has it: by its workgroups a CU and K."""
    tiles = -(-n // 64)
    cells = 4 * tiles * -(-m // 16)
    if cells <= 2 * CUS or (m <= 4 and cells <= 3 * CUS):
        return "cells"
    if m <= 32 or tiles * -(-m // 32) <= 3 * CUS // 2:
        return "rows"
    medium, large = -(-m // 128) * -(-tiles // 4), -(-m // 128) * -(-tiles // 8)
    if medium <= CUS // 2:
        return "halves"
    rest = medium % (2 * CUS)
    two = medium // (2 * CUS) * 17 + (0 if rest == 0 else 12 if rest <= CUS else 17)
    return "large" if k > 2048 and -(-large // CUS) * 16 <= two else "medium"


# (form, m, n, k); n fills whole 16 bytes of 16-bit outputs, n - 1 does not and takes the same form; rows of 2177
# codes are copied, the others read as they lie
CASES = {
    "halves": ("halves", 333, 2232, 1104),
    "medium": ("medium", 1029, 4104, 2208),              # 153 tiles of 128 x 256, one a workgroup
    "medium, tiles in turn": ("medium", 3000, 6000, 2177),  # 576 tiles by 512 workgroups
    "medium, short sums": ("medium", 5000, 4480, 336),   # 720
    "large": ("large", 1900, 5200, 2208),                # 165 tiles of 128 x 512
    "large, tiles in turn": ("large", 3000, 8648, 2192),  # 408 by 256 workgroups
}


@functools.lru_cache(maxsize=1)
def _operands(case):
    """Codes, weight, scales and the exact sums of a case; the last column is the odd one out."""
    form, m, n, k = CASES[case]
    assert _form(m, n, k) == _form(m, n - 1, k) == form
    g = torch.Generator(device=DEV).manual_seed(n)
    codes = torch.randint(-128, 128, (m, k), generator=g, device=DEV, dtype=torch.int8)
    q = torch.randint(-128, 128, (n, k), generator=g, device=DEV, dtype=torch.int8)
    rs = (0.5 + torch.rand(m, generator=g, device=DEV)) / 64
    s = (0.5 + torch.rand(n, generator=g, device=DEV)) / (64 * k ** 0.5)
    sums = codes.double() @ q.double().t().contiguous()
    return codes, q, rs, s, sums


def _check(got, sums, rs, s, residual=None):
    product = sums * rs.double().unsqueeze(1) * s.double()
    want = product if residual is None else product + residual.double()
    slack = 3 * 2.0 ** -24 * product.abs() + 2.0 ** -24 * want.abs()
    limit = slack + HALF[got.dtype] * (want.abs() + slack) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    worst = ((got.double() - want).abs() / limit).max().item()
    assert worst <= 1.0, f"error / bound = {worst:.3f}"


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_tiles(case, whole, dtype):
    """With and without a residual; the first rows have the same bits by the kernels for few rows."""
    codes, q, rs, s, sums = _operands(case)
    n = len(s) if whole else len(s) - 1
    weight = ops.Weight8(q[:n], s[:n])
    res = torch.randn(len(rs), n, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    with torch.inference_mode():
        for residual in (None, res):
            got = ops.linear8(ops.Rows8(codes, rs), weight, residual, dtype=dtype)
            _check(got, sums[:, :n], rs, s[:n], residual)
            for m in (1, 30):
                assert _form(m, n, 1) in ("cells", "rows")
                few = ops.linear8(ops.Rows8(codes[:m], rs[:m]), weight, None if residual is None else residual[:m],
                                  dtype=dtype)
                assert torch.equal(few, got[:m])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("case", ["halves", "medium", "medium, tiles in turn", "large, tiles in turn"])
def test_strided_operands(case, whole, dtype):
    """Codes in rows apart, with other codes behind K, on 16-byte boundaries and not; out and residual in rows
    apart; out as the residual; rows behind the last and columns beside them as they were; a row whose scale is
    NaN, and no other, is NaN."""
    codes, q, rs, s, sums = _operands(case)
    m, k = codes.shape
    side, n = (8, len(s)) if whole else (5, len(s) - 1)
    weight = ops.Weight8(q[:n], s[:n])
    bad = rs.clone()
    bad[m // 2] = float("nan")
    keep = [i for i in range(m) if i != m // 2]
    res = torch.randn(m, n, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(dtype)
    for at, ld in ((0, -(-k // 64) * 64 + 64), (5, k + 37)):
        base = torch.full((m, ld), 77, dtype=torch.int8, device=DEV)
        base[:, at:at + k] = codes
        rows = ops.Rows8(base[:, at:at + k], bad)
        out = torch.full((m + 3, n + 2 * side), 7.0, dtype=dtype, device=DEV)
        held = torch.full((m + 3, n + 2 * side), 9.0, dtype=dtype, device=DEV)
        held[:m, side:side + n] = res
        with torch.inference_mode():
            back = ops.linear8(rows, weight, held[:m, side:side + n], out=out[:m, side:side + n])
            assert back.data_ptr() == out[:m, side:side + n].data_ptr()
            assert torch.isnan(back[m // 2]).all()
            _check(back[keep], sums[keep, :n], rs[keep], s[:n], res[keep])
            ops.linear8(rows, weight, held[:m, side:side + n], out=held[:m, side:side + n])
            assert torch.equal(held[:m, side:side + n][keep], back[keep])
        for t, fill in ((out, 7), (held, 9)):
            assert (t[m:] == fill).all() and (t[:, :side] == fill).all() and (t[:, side + n:] == fill).all()


@pytest.mark.parametrize("case", ["halves", "medium", "large"])
def test_the_longest_sums(case):
    """K = 131071 products of -128 and -128: 2^31 - 16384, the greatest sum there is, exactly."""
    form, m, n, _ = CASES[case]
    k = _hip.LINEAR8_MAX_K
    assert _form(m, n, k) == ("large" if case == "large" else form)
    codes = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    weight = ops.Weight8(torch.full((n, k), -128, dtype=torch.int8, device=DEV), torch.ones(n, device=DEV))
    with torch.inference_mode():
        got = ops.linear8(ops.Rows8(codes, torch.ones(m, device=DEV)), weight, dtype=F32)
    assert (got == float(k * 16384)).all()


def test_graphs():
    """Captured calls of the tile kernels, one with its copy of unaligned codes, replayed in turn on new codes."""
    g = torch.Generator(device=DEV).manual_seed(3)
    held = []
    with torch.inference_mode():
        for case in ("halves", "medium, tiles in turn", "large"):
            codes, q, rs, s, _ = _operands(case)
            static, weight = codes.clone(), ops.Weight8(q, s)
            ops.linear8(ops.Rows8(static, rs), weight)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = ops.linear8(ops.Rows8(static, rs), weight)
            held.append((graph, static, rs, weight, out))
        for _ in range(3):
            for _, static, *_ in held:
                static.copy_(torch.randint(-128, 128, static.shape, generator=g, device=DEV, dtype=torch.int8))
            for graph, *_ in held:
                graph.replay()
            torch.cuda.synchronize()
            for _, static, rs, weight, out in held:
                assert torch.equal(out, ops.linear8(ops.Rows8(static, rs), weight))
