"""8-bit rows and weights without a GPU: layouts, rounding, refusals, the C entry points' checks."""

from __future__ import annotations

import copy
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
from mamba3_amd import Mamba3, _hip, ops

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("libmamba3_hip.so is not built (run __graft_entry__.build())")
    return _hip.load()


def _parts(n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8), torch.rand(n, generator=g)


@pytest.mark.parametrize("n,k", [(1, 1), (64, 128), (65, 129), (150, 200), (63, 64)])
def test_layout_is_the_header_s(n, k):
    codes, scales = _parts(n, k)
    weight = ops.Weight8(codes, scales)
    tn, tk = -(-n // 64), 2 * -(-k // 128)
    assert weight.q.shape == (tn, tk, 4, 64, 16) and weight.scales.shape == (64 * tn,)
    wide = torch.zeros(64 * tn, 64 * tk, dtype=torch.int8)
    wide[:n, :k] = codes
    wide = wide.view(tn, 64, tk, 64)
    for j in range(4):
        for lane in range(64):
            row = 32 * (j // 2) + 8 * (lane % 16 // 4) + 4 * (j % 2) + lane % 4
            col = 16 * (lane // 16)
            assert torch.equal(weight.q[:, :, j, lane], wide[:, row, :, col:col + 16])
    assert torch.equal(weight.scales[:n], scales) and not weight.scales[n:].any()
    assert torch.equal(weight.dequantize(), codes.float() * scales.unsqueeze(1))
    assert torch.equal(weight.dequantize(BF16), (codes.float() * scales.unsqueeze(1)).to(BF16))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_quantize8(dtype):
    """Within half a code, and the ends of the range are codes 127; ties go to even."""
    weight = torch.randn(20, 300, generator=torch.Generator().manual_seed(1)).to(dtype)
    weight[3] = 0
    weight[4, :4] = torch.tensor([127.0, 2.5, -3.5, 63.5]).to(dtype)
    weight[4, 4:] = 0
    held = ops.quantize8(weight)
    most = weight.double().abs().amax(1)
    q = held.q.view(1, 6, 2, 2, 4, 4, 4, 16).permute(0, 2, 5, 3, 6, 1, 4, 7).reshape(64, 384)
    error = (q[:20, :300].double() * most.unsqueeze(1) / 127 - weight.double()).abs()
    assert (error <= most.unsqueeze(1) / 254 * (1 + 1e-12)).all()
    assert q.abs().amax(1)[:20].tolist() == [0 if i == 3 else 127 for i in range(20)]
    assert q[4, :4].tolist() == [127, 2, -4, 64] and not held.dequantize()[3].any()


def test_rows8_takes_codes_as_they_are():
    codes, scales = _parts(6, 64)
    rows = ops.Rows8(codes, scales)
    assert rows.codes.data_ptr() == codes.data_ptr() and rows.shape == (6, 64)
    wide, _ = _parts(6, 96)
    view = ops.Rows8(wide[:, :50], scales)
    assert view.codes.data_ptr() == wide.data_ptr() and view._ld == 96
    for given in (wide[:, 3:53], wide[:, ::2], wide[:, :48].t().contiguous().t(), _parts(6, 33)[0],
                  wide[:1].expand(6, 96), wide.flatten()[:300].as_strided((6, 90), (40, 1))):
        held = ops.Rows8(given, scales)
        assert torch.equal(held.codes, given) and held.codes.stride(1) == 1
        assert held._block() == (held.codes.data_ptr(), held.codes.stride(0), held.scales.data_ptr())
        as_is = given.stride(1) == 1 and given.stride(0) >= given.shape[1]
        assert (held.codes.data_ptr() == given.data_ptr()) == as_is
    cube = ops.Rows8(codes.view(2, 3, 64).transpose(0, 1), scales.view(2, 3).t())
    assert torch.equal(cube.codes, codes.view(2, 3, 64).transpose(0, 1)) and cube.shape == (3, 2, 64)
    assert torch.equal(cube.dequantize(), cube.codes.float() * scales.view(2, 3).t().unsqueeze(-1))
    one = ops.Rows8(codes[2], scales[2])
    assert one.shape == (64,) and torch.equal(one.dequantize(BF16), (codes[2] * scales[2]).to(BF16))
    none = ops.Rows8(codes[:0], scales[:0])
    assert none.shape == (0, 64)
    twin = copy.deepcopy(view)
    assert torch.equal(twin.codes, view.codes) and twin._block()[0] == twin.codes.data_ptr() != view._block()[0]


@pytest.mark.parametrize("make,message", [
    (lambda c, s: ops.Rows8(c.int(), s), "codes must"),
    (lambda c, s: ops.Rows8(c[:, :0], s), "codes must"),
    (lambda c, s: ops.Rows8(c, s[:3]), "scales must"),
    (lambda c, s: ops.Rows8(c, s.double()), "scales must"),
    (lambda c, s: ops.Rows8(torch.zeros(1, 131072, dtype=torch.int8), s[:1]), "at most 131071"),
    (lambda c, s: ops.Rows8(c, s.to("meta")), "same device"),
    (lambda c, s: ops.Weight8(c[0], s), "codes must"),
    (lambda c, s: ops.Weight8(c[:0], s[:0]), "codes must"),
    (lambda c, s: ops.Weight8(c.short(), s), "codes must"),
    (lambda c, s: ops.Weight8(c, s.half()), "scales must"),
    (lambda c, s: ops.Weight8(c, s[:2]), "scales must"),
    (lambda c, s: ops.Weight8(c, s.to("meta")), "same device"),
    (lambda c, s: ops.Weight8(torch.zeros(1, 131072, dtype=torch.int8), s[:1]), "at most 131071"),
    (lambda c, s: ops.quantize8(c), "floating"),
    (lambda c, s: ops.quantize8(s), "floating"),
    (lambda c, s: ops.quantize8(torch.full((2, 3), float("nan"))), "NaN"),
    (lambda c, s: ops.quantize8(torch.full((2, 3), float("inf"))), "infinities"),
    (lambda c, s: ops.quantize8_rows(c), "x must"),
    (lambda c, s: ops.quantize8_rows(s[0]), "x must"),
    (lambda c, s: ops.quantize8_rows(s.double()), "x must"),
    (lambda c, s: ops.quantize8_rows(s[:0]), "rows of 0"),
    (lambda c, s: ops.quantize8_rows(torch.zeros(131072)), "rows of 131072"),
    (lambda c, s: ops.rms_norm8(s, s[:3]), "weight must"),
    (lambda c, s: ops.rms_norm8(s, s.double()), "weight must"),
    (lambda c, s: ops.rms_norm8(s, s, add=s[:1]), "add must"),
    (lambda c, s: ops.rms_norm8(s.half(), s, add=s), "add must"),
    (lambda c, s: ops.rms_norm8(s, s, keep_sum=True), "needs add"),
    (lambda c, s: ops.rms_norm8(s, s, -1.0), "eps"),
    (lambda c, s: ops.rms_norm8(s, s, float("nan")), "eps"),
    (lambda c, s: ops.linear8(ops.Rows8(c, s), ops.Weight8(c[:, :60], s)), "do not fit"),
    (lambda c, s: ops.linear8(ops.Rows8(c, s), ops.Weight8(c, s), dtype=torch.float64), "dtype must"),
    (lambda c, s: ops.linear8(ops.Rows8(c, s), ops.Weight8(c, s), torch.zeros(8, 7)), "residual must"),
    (lambda c, s: ops.linear8(ops.Rows8(c, s), ops.Weight8(c, s), out=torch.zeros(7, 8)), "out must"),
    (lambda c, s: ops.linear8(ops.Rows8(c, s), ops.Weight8(c, s), torch.zeros(8, 8), dtype=BF16),
     "residual must"),
])
def test_refusals(make, message):
    with pytest.raises(ValueError, match=message):
        make(*_parts(8, 64))


def test_off_the_gpu_and_under_autograd():
    codes, scales = _parts(8, 64)
    x, weight = torch.zeros(8, 64), ops.Weight8(codes, scales)
    for call in (lambda: ops.quantize8_rows(x), lambda: ops.rms_norm8(x, x[0]),
                 lambda: ops.linear8(ops.Rows8(codes, scales), weight)):
        with pytest.raises(RuntimeError, match="ROCm devices only"):
            call()
    trained = ops.Rows8(codes, torch.rand(8, requires_grad=True))
    with pytest.raises(RuntimeError, match="no backward"):
        trained.dequantize()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for call in (lambda: ops.quantize8_rows(dual), lambda: ops.rms_norm8(x, x[0], add=dual),
                     lambda: ops.linear8(ops.Rows8(codes, scales), weight, dual[:, :8])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def _rows_args(rows=4, dim=100, stride=112):
    return _hip.Rows8Args(rows, dim, 1e-5, 0, _hip.Tensor(0x100000, _hip.F32, 0, (dim, 1)),
                          codes=0x200000, codes_stride=stride, scales=0x300000)


def test_rows8_is_checked_on_the_host(lib):
    call = lib.m3_rows8
    assert call(None, None) == 1 and b"NULL" in lib.m3_last_error()
    assert call(ctypes.byref(_rows_args(rows=0)), None) == 0
    weight = _hip.Tensor(0x400000, _hip.BF16, 0, (1,))
    add = _hip.Tensor(0x500000, _hip.F16, 0, (100, 1))
    for changes, code, text in (
            (dict(rows=-1), 1, b"negative"), (dict(rows=1 << 30), 2, b"below 2^30"),
            (dict(dim=131072), 2, b"at most 131071"), (dict(dim=0), 2, b"dim 0"),
            (dict(x=_hip.Tensor()), 1, b"x: required"),
            (dict(x=_hip.Tensor(0x100000, 7, 0, (100, 1))), 1, b"x: invalid dtype"),
            (dict(x=_hip.Tensor(0x100002, _hip.F32, 0, (100, 1))), 1, b"x: pointer"),
            (dict(x=_hip.Tensor(0x100000, _hip.F32, 0, (200, 2))), 2, b"x: innermost"),
            (dict(x=_hip.Tensor(0x100000, _hip.F32, 0, (-100, 1))), 2, b"x: negative"),
            (dict(codes=None), 1, b"NULL"), (dict(scales=None), 1, b"NULL"),
            (dict(codes=0x200008), 2, b"aligned"), (dict(codes_stride=100), 2, b"aligned"),
            (dict(scales=0x300002), 2, b"aligned"), (dict(codes_stride=96), 1, b"overlap"),
            (dict(add=add), 1, b"add needs weight"),
            (dict(weight=weight, sum_out=add), 2, b"sum_out: dtype"),
            (dict(weight=weight, sum_out=_hip.Tensor(0x600000, _hip.F32, 0, (100, 1))), 1, b"needs add"),
            (dict(weight=weight, eps=-1.0), 1, b"eps"), (dict(weight=weight, eps=float("nan")), 1, b"eps"),
            (dict(weight=weight, add=add, sum_out=_hip.Tensor(0x600000, _hip.F32, 0, (50, 1))), 1, b"rows of"),
            (dict(codes=0x100000 + 3 * 400 + 384), 1, b"overlap another"),
            (dict(scales=0x100000), 1, b"overlap another"), (dict(scales=0x200000 + 3 * 112 + 108), 1, b"overlap s"),
            (dict(weight=weight, add=add, codes=0x500000), 1, b"overlap another"),
            (dict(weight=weight, add=add, codes=0x400000), 1, b"overlap another"),
            (dict(weight=weight, add=add, sum_out=_hip.Tensor(0x100004, _hip.F32, 0, (100, 1))), 1, b"without being"),
            (dict(weight=weight, add=add, sum_out=_hip.Tensor(0x100000, _hip.F32, 0, (104, 1))), 1, b"without being"),
            (dict(weight=weight, add=add, sum_out=_hip.Tensor(0x500000, _hip.F32, 0, (100, 1))), 1, b"without being"),
            (dict(weight=weight, add=add, sum_out=_hip.Tensor(0x3ffffc, _hip.F32, 0, (100, 1))), 1, b"without being")):
        args = _rows_args()
        for field, value in changes.items():
            setattr(args, field, value)
        assert call(ctypes.byref(args), None) == code, (changes, lib.m3_last_error())
        assert text in lib.m3_last_error(), (changes, lib.m3_last_error())
    args = _rows_args()
    args.x.dtype, args.weight, args.add = _hip.BF16, weight, add
    assert call(ctypes.byref(args), None) == 2 and b"add: dtype" in lib.m3_last_error()


def _args(m=4, n=64, k=256):
    return _hip.Linear8Args(m, n, k, _hip.BF16, 0, 0x100000, k, 0x200000, 0x300000, 0x400000,
                            out=_hip.Tensor(0x500000, _hip.BF16, 0, (n, 1)))


def test_linear8_s_workspace(lib):
    """Rows of codes that are not aligned, or may not be read past their end, are copied for the
    kernels for many rows."""
    need = ctypes.c_size_t(7)
    query = lib.m3_linear8_workspace_size
    assert query(None, ctypes.byref(need)) == 1 and query(ctypes.byref(_args()), None) == 1
    for m, n, k, at, exact, bytes_ in (
            (4, 64, 256, 0, 0, 0), (4, 64, 250, 0, 0, 0), (4, 64, 256, 3, 1, 0), (5000, 64 * 20, 256, 0, 0, 0),
            (5000, 64 * 20, 256, 0, 1, 0), (5000, 64 * 20, 256, 1, 0, 5000 * 256), (0, 64, 256, 1, 0, 0),
            (5000, 64 * 20, 250, 0, 0, 5000 * 256), (4, 64 * 20, 250, 0, 1, 0)):
        args = _args(m, n, k)
        args.codes, args.exact, args.out.ptr, args.q = (1 << 40) + at, exact, 1 << 41, 1 << 42
        assert query(ctypes.byref(args), ctypes.byref(need)) == 0 and need.value == bytes_, (m, n, k, at)
    args = _args(5000, 64 * 20, 250)
    args.codes, args.out.ptr, args.q = 1 << 40, 1 << 41, 1 << 42
    for ws, size in ((None, 5000 * 256), (1 << 43, 5000 * 256 - 1), ((1 << 43) + 8, 5000 * 256)):
        args.workspace, args.workspace_bytes = ws, size
        assert lib.m3_linear8(ctypes.byref(args), None) == 4 and b"workspace of 1280000" in lib.m3_last_error()
    args.workspace, args.workspace_bytes = (1 << 41) + 64, 5000 * 256
    assert lib.m3_linear8(ctypes.byref(args), None) == 1 and b"overlaps the workspace" in lib.m3_last_error()


def test_linear8_is_checked_on_the_host(lib):
    call = lib.m3_linear8
    assert call(None, None) == 1 and b"NULL" in lib.m3_last_error()
    assert call(ctypes.byref(_args(m=0)), None) == 0 and call(ctypes.byref(_args(n=0)), None) == 0
    for changes, code, text in (
            (dict(m=-1), 1, b"negative"), (dict(m=1 << 30), 2, b"below 2^30"),
            (dict(n=(1 << 27) + 1), 2, b"2^27"), (dict(k=131072), 2, b"131071"), (dict(k=0), 2, b"K = 0"),
            (dict(dtype=5), 1, b"dtype"), (dict(codes=None), 1, b"NULL"), (dict(row_scales=None), 1, b"NULL"),
            (dict(q=None), 1, b"NULL"), (dict(scales=None), 1, b"NULL"),
            (dict(q=0x300008), 2, b"aligned"), (dict(scales=0x400004), 2, b"aligned"),
            (dict(row_scales=0x200002), 2, b"aligned"), (dict(codes_stride=240), 2, b"codes_stride 240"),
            (dict(codes_stride=(1 << 22) + 16), 2, b"codes_stride"),
            (dict(out=_hip.Tensor()), 1, b"out: required"),
            (dict(out=_hip.Tensor(0x500000, _hip.F32, 0, (64, 1))), 2, b"out: dtype"),
            (dict(out=_hip.Tensor(0x500000, _hip.BF16, 0, (32, 1))), 1, b"rows of out"),
            (dict(out=_hip.Tensor(0x1003fe, _hip.BF16, 0, (64, 1))), 1, b"out overlaps codes"),
            (dict(out=_hip.Tensor(0x20000e, _hip.BF16, 0, (64, 1))), 1, b"out overlaps codes"),
            (dict(out=_hip.Tensor(0x303ffe, _hip.BF16, 0, (64, 1))), 1, b"out overlaps codes"),
            (dict(out=_hip.Tensor(0x4000fe, _hip.BF16, 0, (64, 1))), 1, b"out overlaps codes"),
            (dict(residual=_hip.Tensor(0x500010, _hip.BF16, 0, (64, 1))), 1, b"residual without"),
            (dict(residual=_hip.Tensor(0x500000, _hip.BF16, 0, (72, 1))), 1, b"residual without")):
        args = _args()
        for field, value in changes.items():
            setattr(args, field, value)
        assert call(ctypes.byref(args), None) == code, (changes, lib.m3_last_error())
        assert text in lib.m3_last_error(), (changes, lib.m3_last_error())


def test_rows8_values_is_checked_on_the_host(lib):
    call = lib.m3_rows8_values

    def block(rows=4):
        return _hip.Rows8ValuesArgs(rows, 100, 0x100000, 112, 0x200000, _hip.Tensor(0x300000, _hip.BF16, 0, (100, 1)))

    assert call(None, None) == 1 and b"NULL" in lib.m3_last_error()
    assert call(ctypes.byref(block(0)), None) == 0
    for changes, code, text in (
            (dict(rows=-1), 1, b"negative"), (dict(rows=1 << 30), 2, b"below 2^30"),
            (dict(dim=131072), 2, b"at most 131071"), (dict(dim=0), 2, b"dim 0"),
            (dict(codes=None), 1, b"NULL"), (dict(scales=None), 1, b"NULL"),
            (dict(scales=0x200001), 2, b"aligned"), (dict(codes_stride=96), 1, b"overlap"),
            (dict(out=_hip.Tensor()), 1, b"out: required"),
            (dict(out=_hip.Tensor(0x300000, _hip.BF16, 0, (200, 2))), 2, b"out: innermost"),
            (dict(out=_hip.Tensor(0x300000, _hip.BF16, 0, (99, 1))), 1, b"rows of out"),
            (dict(out=_hip.Tensor(0x100000 + 3 * 112 + 98, _hip.BF16, 0, (100, 1))), 1, b"out overlaps"),
            (dict(out=_hip.Tensor(0x20000e, _hip.BF16, 0, (100, 1))), 1, b"out overlaps")):
        args = block()
        for field, value in changes.items():
            setattr(args, field, value)
        assert call(ctypes.byref(args), None) == code, (changes, lib.m3_last_error())
        assert text in lib.m3_last_error(), (changes, lib.m3_last_error())


def test_structs_match_the_header_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    pairs = (("m3_rows8_args", _hip.Rows8Args, _hip.ROWS8), ("m3_linear8_args", _hip.Linear8Args, _hip.LINEAR8),
             ("m3_rows8_values_args", _hip.Rows8ValuesArgs, _hip.ROWS8_VALUES))
    lines = ['#include "mamba3_hip.h"', "#include <stdio.h>", "int main(void) {",
             'printf("max - %d\\n", M3_LINEAR8_MAX_K);']
    for name, py, _ in pairs:
        lines.append(f'printf("{name} - %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    source = tmp_path / "layout.c"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{os.path.join(ROOT, 'include')}", str(source), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True)
    structs = {name: py for name, py, _ in pairs}
    for line in out.stdout.splitlines():
        name, field, value = line.split()
        if name == "max":
            assert _hip.LINEAR8_MAX_K == int(value)
            continue
        size = ctypes.sizeof(structs[name]) if field == "-" else getattr(structs[name], field).offset
        assert size == int(value), line
    for _, py, packed in pairs:
        assert packed.size == ctypes.sizeof(py)


def test_quantize_prefill_holds_copies_and_changes_nothing():
    model = Mamba3(64, depth=2).to(BF16)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    assert model.quantize_prefill() is model
    assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items())
    assert list(model.state_dict()) == list(before)
    mixer = model.layers[1].mixer
    for name in ("in_proj", "out_proj"):
        weight = getattr(mixer, name).weight
        want = ops.quantize8(weight)
        assert torch.equal(mixer._weight8(name).q, want.q)
        assert torch.equal(mixer._weight8(name).scales, want.scales)
    with pytest.raises(RuntimeError, match="ROCm devices only"), torch.no_grad():
        model(torch.zeros(1, 2, 64, dtype=BF16))
    model.load_state_dict(before)
    with pytest.raises(RuntimeError, match="quantize_prefill; call it again"):
        mixer._weight8("in_proj")
    with pytest.raises(RuntimeError, match="quantize_prefill; call it again"), torch.no_grad():
        model(torch.zeros(1, 2, 64, dtype=BF16))


def test_quantize_prefill_and_quantize_decode():
    """The 4-bit copies' rounding changes the weights: the 8-bit ones are made after it."""
    model = Mamba3(64, depth=1).to(BF16).quantize_prefill().quantize_decode(32)
    mixer = model.layers[0].mixer
    with pytest.raises(RuntimeError, match="call it again"):
        mixer._weight8("out_proj")
    model.quantize_prefill()
    assert mixer._weight8("out_proj") is not None and mixer._weight4("out_proj") is not None


def test_quantize_prefill_holds_every_layer_or_none():
    model = Mamba3(64, depth=2)
    with torch.no_grad():
        model.layers[1].mixer.out_proj.weight[3, 5] = float("inf")
    with pytest.raises(ValueError, match="infinities"):
        model.quantize_prefill()
    assert not any(layer.mixer._prefill8 for layer in model.layers)
    with torch.inference_mode():
        unversioned = Mamba3(64, depth=1)
        with pytest.raises(ValueError, match="inference_mode"):
            unversioned.quantize_prefill()


def test_a_graph_decoder_sees_copies_made_after_it():
    """A graph of more rows than the decode kernels' runs on the projections that it was captured with: one from
    before ``quantize_prefill`` is not the model's step any more. (Checked on a decoder without its capture.)"""
    from mamba3_amd.model import _HipGraphDecoder, _layers_in8, _storage_signature

    def decoder_for(model, rows):
        dec = object.__new__(_HipGraphDecoder)
        dec.model, dec._in8 = model, _layers_in8(model, rows)
        dec._captured = [_storage_signature(w) for w in model.parameters()]
        return dec

    model = Mamba3(16, d_state=8, depth=2)
    few, many = decoder_for(model, ops.DECODE_LINEAR_ROWS), decoder_for(model, ops.DECODE_LINEAR_ROWS + 1)
    few.validate(), many.validate()
    model.quantize_prefill()
    few.validate()
    with pytest.raises(RuntimeError, match="recreate"):
        many.validate()
    many = decoder_for(model, 200)
    model.quantize_prefill()  # of the same weights: the same copies
    many.validate(), few.validate()


def test_linear8_s_workspace_overlaps_nothing(lib):
    """The copy of the codes would be written over what the call reads."""
    m, n, k = 5000, 64 * 20, 250
    size = m * 256

    def block(workspace):
        args = _args(m, n, k)
        args.codes, args.out.ptr, args.q, args.residual = 1 << 40, 1 << 41, 1 << 42, _hip.Tensor(1 << 44, _hip.BF16, 0, (n, 1))
        args.row_scales, args.scales = 1 << 45, 1 << 46
        args.workspace, args.workspace_bytes = workspace, size
        return args

    need = ctypes.c_size_t(0)
    for at, bytes_, text in ((1 << 40, (m - 1) * k + k, b"codes"), (1 << 41, m * n * 2, b"out"),
                             (1 << 42, 20 * 4 * 4096, b"the weight"), (1 << 44, m * n * 2, b"residual"),
                             (1 << 45, m * 4, b"scales"), (1 << 46, n * 4, b"scales")):
        for workspace in (at, at - size + 16, (at + bytes_ - 1) // 16 * 16):
            args = block(workspace)
            assert lib.m3_linear8_workspace_size(ctypes.byref(args), ctypes.byref(need)) == 1, hex(workspace)
            assert b"overlaps the workspace" in lib.m3_last_error() and text in lib.m3_last_error()
        for workspace in (at - size, (at + bytes_ + 15) // 16 * 16):
            args = block(workspace)
            assert lib.m3_linear8_workspace_size(ctypes.byref(args), ctypes.byref(need)) == 0, hex(workspace)
            assert need.value == size
    args = block(1 << 40)  # not used, and so not looked at, where nothing is copied
    args.codes_stride = 256
    assert lib.m3_linear8_workspace_size(ctypes.byref(args), ctypes.byref(need)) == 0 and need.value == 0


def test_models_pickled_before_there_were_copies():
    """A mixer whose state lacks the dicts of copies is one without any."""
    mixer = Mamba3(64, depth=1).layers[0].mixer
    for name in ("_decode4", "_prefill8"):
        del mixer.__dict__[name]
    twin = copy.deepcopy(mixer)
    model = Mamba3(64, depth=1)
    model.layers[0].mixer = twin
    assert twin._weight8("in_proj") is None and twin._weight4("out_proj") is None
    with pytest.raises(RuntimeError, match="ROCm devices only"), torch.no_grad():
        model(torch.zeros(1, 2, 64))
    with pytest.raises(RuntimeError, match="ROCm devices only"), torch.no_grad():
        model.step(torch.zeros(70, 1, 64))
    model.quantize_prefill()
    assert twin._weight8("in_proj") is not None
    assert mixer._weight8("in_proj") is None and Mamba3(64, depth=1).layers[0].mixer._prefill8 == {}
