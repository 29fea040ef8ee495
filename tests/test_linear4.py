"""4-bit weights without a GPU: the tile layout, quantisation, refusals, the C entry point's checks."""

from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
from mamba3_amd import Mamba3, _hip, ops


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("libmamba3_hip.so is not built (run __graft_entry__.build())")
    return _hip.load()


def _parts(n, k, group, zeros=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.rand(n, k // group, generator=g).to(torch.float16)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return packed, scales, z


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (37, 160, 32), (50, 192, 64)])
def test_layout_is_the_header_s(n, k, group, zeros):
    packed, scales, z = _parts(n, k, group, zeros)
    weight = ops.Weight4(packed, scales, z)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1)
    tn, tk, per = -(-n // 16), -(-k // 128), 128 // group
    assert weight.codes.shape == (tn, tk, 64, 4, 4)
    word = sum(weight.codes[..., b].long() << (8 * b) for b in range(4))
    for lane in range(64):
        for i in range(4):
            for e in range(8):
                got = word[:, :, lane, i] >> (4 * (e // 2) + 16 * (e % 2)) & 15
                for t in range(tn):
                    for u in range(tk):
                        row, col = 16 * t + lane % 16, 128 * u + 32 * i + 8 * (lane // 16) + e
                        assert got[t, u] == (codes[row, col] if row < n and col < k else 0)
    for held, given in ((weight.scales, scales), (weight.zeros, z)):
        if given is None:
            assert held is None
            continue
        assert held.shape == (tn, tk, per, 16)
        wide = held.permute(0, 3, 1, 2).reshape(16 * tn, tk * per)
        assert torch.equal(wide[:n, :k // group], given)
        assert not wide[n:].any() and not wide[:, k // group:].any()


@pytest.mark.parametrize("zeros", [True, False])
def test_dequantize(zeros):
    packed, scales, z = _parts(37, 160, 32, zeros)
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1).float().view(37, -1, 32)
    shift = z.float().unsqueeze(-1) if zeros else 8.0
    want = ((codes - shift) * scales.float().unsqueeze(-1)).flatten(1)
    weight = ops.Weight4(packed, scales, z)
    assert torch.equal(weight.dequantize(torch.float32), want)
    assert torch.equal(weight.dequantize(), want.half())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize4_is_within_half_a_step(group, zeros, dtype):
    """A value lies within half a step of its code's, or within what the scale's own rounding
    (half a step of its type, times 15 codes) moves the ends of the range, plus the zero's half."""
    g = torch.Generator().manual_seed(group)
    weight = torch.randn(24, 384, generator=g).to(dtype)
    weight[3] = 0
    weight[4] = weight[4].abs()
    held = ops.quantize4(weight, group, zeros=zeros)
    assert held.shape == (24, 384) and held.group == group
    w = weight.float().unflatten(1, (-1, group))
    step = ((w.amax(-1).clamp(min=0) - w.amin(-1).clamp(max=0)) / 15 if zeros else
            torch.maximum(w.amax(-1) / 7, -w.amin(-1) / 8)).unsqueeze(-1)
    error = (held.dequantize(torch.float32).unflatten(1, (-1, group)) - w).abs()
    half = 2.0 ** -8 if held.dtype == torch.bfloat16 else 2.0 ** -11
    assert (error <= step * ((1.0 if zeros else 0.5) + 15 * half) * (1 + half)).all()
    assert not held.dequantize()[3].any()


def test_quantize4_twice_is_the_same_weight():
    weight = torch.randn(16, 256, generator=torch.Generator().manual_seed(1))
    once = ops.quantize4(weight, 64, zeros=False).dequantize(torch.float32)
    # codes that reach neither end do not come back as such: hold the range with both ends
    weight[:, 0::64], weight[:, 1::64] = -4.0, 3.5
    once = ops.quantize4(weight, 64, zeros=False).dequantize(torch.float32)
    assert torch.equal(ops.quantize4(once, 64, zeros=False).dequantize(torch.float32), once)


@pytest.mark.parametrize("make,message", [
    (lambda p, s, z: ops.Weight4(p.int(), s, z), "packed must"),
    (lambda p, s, z: ops.Weight4(p[0], s, z), "packed must"),
    (lambda p, s, z: ops.Weight4(p, s[:3], z), "scales must"),
    (lambda p, s, z: ops.Weight4(p, s.float(), z), "bfloat16 or float16"),
    (lambda p, s, z: ops.Weight4(p, s[:, :1], None), "groups must"),
    (lambda p, s, z: ops.Weight4(p, s, z[:, :1]), "zeros must"),
    (lambda p, s, z: ops.Weight4(p, s, z.int()), "zeros must"),
    (lambda p, s, z: ops.quantize4(torch.zeros(4, 100), 64), "multiple of group"),
    (lambda p, s, z: ops.quantize4(torch.zeros(4, 96), 48), "multiple of group"),
    (lambda p, s, z: ops.quantize4(torch.zeros(4, 128, dtype=torch.int32)), "floating"),
    (lambda p, s, z: ops.quantize4(torch.full((4, 128), float("nan"))), "NaN"),
    (lambda p, s, z: ops.quantize4(torch.full((4, 128), 3e38), dtype=torch.float16), "range"),
    (lambda p, s, z: ops.quantize4(torch.zeros(4, 128), dtype=torch.float32), "bfloat16 or"),
])
def test_weight_refusals(make, message):
    with pytest.raises(ValueError, match=message):
        make(*_parts(8, 256, 64))


def test_linear4_refusals():
    weight = ops.Weight4(*_parts(8, 256, 64))
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    assert not ops.linear4_supported(x, weight)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        ops.linear4(x, weight)


def test_quantize_decode_refusals():
    with pytest.raises(ValueError, match="16 weights"):
        Mamba3(64, depth=1).quantize_decode()
    with pytest.raises(ValueError, match="causal"):
        Mamba3(64, depth=1, causal=False).to(torch.bfloat16).quantize_decode(32)
    model = Mamba3(64, depth=1).to(torch.bfloat16)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    for group in (128, 48):
        with pytest.raises(ValueError, match="group must"):
            model.quantize_decode(group)
    assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items())
    assert model.quantize_decode(32) is model
    assert list(model.state_dict()) == list(before)
    mixer = model.layers[0].mixer
    assert torch.equal(mixer.in_proj.weight, mixer._weight4("in_proj").dequantize(torch.bfloat16))
    model.load_state_dict(before)
    with pytest.raises(RuntimeError, match="call it again"):
        mixer._weight4("in_proj")


def test_quantize_decode_changes_every_layer_or_none():
    model = Mamba3(64, depth=2).to(torch.bfloat16)
    with torch.no_grad():
        model.layers[1].mixer.out_proj.weight[3, 5] = float("nan")
    before = model.layers[0].mixer.in_proj.weight.clone()
    with pytest.raises(ValueError, match="NaN"):
        model.quantize_decode(32)
    assert torch.equal(model.layers[0].mixer.in_proj.weight, before)
    assert all(layer.mixer._weight4("in_proj") is None for layer in model.layers)


def _args(m=4, n=64, k=256):
    return _hip.Linear4Args(m, n, k, _hip.BF16, _hip.F16, 64, 1e-5, 0x100000, 0x200000, 0x300000,
                            _hip.Tensor(0x400000, _hip.BF16, 0, (k, 1)),
                            out=_hip.Tensor(0x500000, _hip.BF16, 0, (n, 1)))


def test_validation_on_the_host(lib):
    call = lib.m3_linear4
    assert call(None, None) == 1 and b"NULL" in lib.m3_last_error()
    assert call(ctypes.byref(_args(m=0)), None) == 0 and call(ctypes.byref(_args(n=0)), None) == 0
    for field, value, code, text in (
            ("m", -1, 1, b"negative"), ("m", 257, 2, b"M = 257"), ("dtype", _hip.F32, 2, b"dtype"),
            ("scale_dtype", _hip.F32, 2, b"scale dtype"), ("group", 48, 2, b"group 48"),
            ("k", 288, 2, b"K = 288"), ("k", 0, 2, b"K = 0"), ("codes", None, 1, b"NULL"),
            ("scales", None, 1, b"NULL"), ("codes", 0x100008, 2, b"aligned"),
            ("scales", 0x200004, 2, b"aligned"), ("zeros", 0x300002, 2, b"aligned")):
        args = _args()
        setattr(args, field, value)
        assert call(ctypes.byref(args), None) == code, field
        assert text in lib.m3_last_error(), field
    for name, field, value, code, text in (
            ("x", "ptr", None, 1, b"x: required"), ("x", "ptr", 0x400008, 2, b"aligned"),
            ("x", "dtype", _hip.F16, 2, b"x: dtype"), ("out", "ptr", None, 1, b"out: required"),
            ("out", "ptr", 0x400100, 1, b"overlaps"), ("out", "ptr", 0x100100, 1, b"overlaps")):
        args = _args()
        setattr(getattr(args, name), field, value)
        assert call(ctypes.byref(args), None) == code, (name, value)
        assert text in lib.m3_last_error(), (name, value)
    args = _args()
    args.residual = _hip.Tensor(0x500000 + 16, _hip.BF16, 0, (64, 1))
    assert call(ctypes.byref(args), None) == 1 and b"residual" in lib.m3_last_error()
    args = _args()
    args.residual = _hip.Tensor(0x500000, _hip.BF16, 0, (72, 1))
    assert call(ctypes.byref(args), None) == 1 and b"residual" in lib.m3_last_error()
    args = _args()
    args.out.stride[0] = 8
    assert call(ctypes.byref(args), None) == 1 and b"rows of out" in lib.m3_last_error()


def test_rows_of_x_too_far_apart_are_refused(lib):
    """Offsets within x, and of the rows of a block past the last, fit 32 bits only up to here."""
    for m, stride in ((17, 1 << 24), (17, (1 << 25) - 64), (2, 1 << 28), (256, 1 << 21)):
        args = _args(m=m, n=6144)
        args.x = _hip.Tensor(1 << 40, _hip.BF16, 0, (stride, 1))
        assert lib.m3_linear4(ctypes.byref(args), None) == 2, (m, stride)
        assert b"512 MB" in lib.m3_last_error(), (m, stride)


def test_struct_matches_the_header_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ['#include "mamba3_hip.h"', "#include <stdio.h>", "int main(void) {",
             'printf("- %zu\\n", sizeof(m3_linear4_args));']
    lines += [f'printf("{f} %zu\\n", offsetof(m3_linear4_args, {f}));'
              for f, _ in _hip.Linear4Args._fields_]
    source = tmp_path / "layout.c"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{os.path.join(ROOT, 'include')}", str(source), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True)
    for line in out.stdout.splitlines():
        field, value = line.split()
        size = (ctypes.sizeof(_hip.Linear4Args) if field == "-"
                else getattr(_hip.Linear4Args, field).offset)
        assert size == int(value), field


def test_the_norm_s_epsilon_and_what_out_overlaps(lib):
    call = lib.m3_linear4
    for eps in (-1e-5, float("nan")):
        args = _args()
        args.norm_weight, args.norm_eps = _hip.Tensor(0x600000, _hip.BF16, 0, (1,)), eps
        assert call(ctypes.byref(args), None) == 1 and b"norm_eps" in lib.m3_last_error()
    # out [4, 64] bf16 over the last bytes of the scales (4 tile rows x 2 x 2 groups x 16, 512 bytes), the
    # zeros (256 bytes) and the norm's weight (512)
    for at, size in ((0x200000, 512), (0x300000, 256), (0x600000, 512)):
        args = _args()
        args.norm_weight = _hip.Tensor(0x600000, _hip.BF16, 0, (1,))
        args.out.ptr = at + size - 2
        assert call(ctypes.byref(args), None) == 1, hex(at)
        assert b"out overlaps" in lib.m3_last_error()
        args.out.ptr = at - (3 * 64 + 64) * 2 + 2
        assert call(ctypes.byref(args), None) == 1, hex(at)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_zeros_above_a_code_are_refused(group):
    """Not held as 15: a format whose zeros are off by one (1..16) would lose weight unnoticed."""
    packed, scales, z = _parts(20, 256, group)
    z[3, -1] = 16
    with pytest.raises(ValueError, match="zeros must be .* 0 to 15"):
        ops.Weight4(packed, scales, z)
    z[3, -1] = 15
    assert ops.Weight4(packed, scales, z).zeros.max() <= 15



def test_quantize_decode_of_a_shared_weight():
    model = Mamba3(64, depth=3).to(torch.bfloat16)
    model.layers[2].mixer.in_proj.weight = model.layers[0].mixer.in_proj.weight
    model.quantize_decode(32)
    for layer in model.layers:
        for name in ("in_proj", "out_proj"):
            assert torch.equal(layer.mixer._weight4(name).dequantize(torch.bfloat16),
                               getattr(layer.mixer, name).weight)



def test_quantize_decode_writes_no_infinity():
    """7 codes times the rounded scale of f16's largest value are above it."""
    model = Mamba3(64, depth=2).half()
    with torch.no_grad():
        model.layers[1].mixer.out_proj.weight[0, 0] = 65504.0
    before = {k: v.clone() for k, v in model.state_dict().items()}
    with pytest.raises(ValueError, match="beyond"):
        model.quantize_decode(32, zeros=False)
    assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items())


def test_quantize_decode_without_versions_changes_nothing():
    """Weights made under inference_mode have no version by which a later change would show."""
    with torch.inference_mode():
        model = Mamba3(64, depth=2).to(torch.bfloat16)
        before = {k: v.clone() for k, v in model.state_dict().items()}
        with pytest.raises(ValueError, match="inference_mode"):
            model.quantize_decode(32)
        assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items())
    assert not any(layer.mixer._decode4 for layer in model.layers)
