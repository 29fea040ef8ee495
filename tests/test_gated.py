"""The gated recurrence without a GPU: the 64-bit oracle's own checks, refusals of ``ops.gated_scan``
/ ``ops.gated_step``, and the C entry points' host-side checks."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from conftest import ROOT  # noqa: F401
from mamba3_amd import _hip, ops
from oracle import gated as og


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_hip.LIB_PATH):
        pytest.skip("libmamba3_hip.so is not built (run __graft_entry__.build())")
    return _hip.load()


def test_oracle_against_the_closed_form():
    """h_t = sum_j exp(S_t - S_j) b_j with S the running sum of log decays."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 20, 3, generator=g, dtype=torch.float64)
    decay = -torch.rand(2, 20, 3, generator=g, dtype=torch.float64)
    y, final = og.scan(x, decay)
    total = decay.cumsum(1)
    want = torch.stack([(torch.exp(total[:, t:t + 1] - total[:, :t + 1]) * x[:, :t + 1]).sum(1)
                        for t in range(20)], 1)
    torch.testing.assert_close(y, want, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(final, want[:, -1], rtol=1e-12, atol=1e-12)


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    args = [torch.randn(2, 5, 3, generator=g, dtype=torch.float64) for _ in range(3)]
    args += [torch.rand(3, generator=g, dtype=torch.float64) + 0.1,
             torch.randn(2, 3, generator=g, dtype=torch.float64)]
    lengths = torch.tensor([5, 3])
    reset = torch.zeros(2, 5, dtype=torch.bool)
    reset[0, 2] = True
    for a in args:
        a.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *a: og.scan(*a, lengths=lengths, reset=reset), args)


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kwargs,message", [
    (dict(x=_x(2, 8)), r"\[B, L, C\]"),
    (dict(decay=_x(2, 5, 4)), "shape of x"),
    (dict(decay=_x(2, 4, 8, dtype=torch.bfloat16)), "share one dtype"),
    (dict(x=_x(2, 4, 8, dtype=torch.float64), decay=_x(2, 4, 8, dtype=torch.float64)),
     "share one dtype"),
    (dict(gate=_x(2, 4, 8)), "together"),
    (dict(rate=_x(8)), "together"),
    (dict(gate=_x(2, 4, 8), rate=_x(4)), "rate must"),
    (dict(gate=_x(2, 4, 8), rate=torch.zeros(8, dtype=torch.int32)), "rate must"),
    (dict(initial_state=_x(2, 4)), "initial_state"),
    (dict(initial_state=_x(2, 8, dtype=torch.bfloat16)), "initial_state"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=_x(2)), "lengths"),
    (dict(reset=torch.zeros(2, 5, dtype=torch.bool)), "reset"),
    (dict(reset=_x(2, 4)), "reset"),
])
def test_scan_refusals(kwargs, message):
    args = dict(x=_x(2, 4, 8), decay=_x(2, 4, 8)) | kwargs
    with pytest.raises(ValueError, match=message):
        ops.gated_scan(**args)


def test_step_refusals():
    x, state = _x(2, 8), _x(2, 8)
    with pytest.raises(ValueError, match=r"\[B, C\]"):
        ops.gated_step(_x(2, 1, 8), _x(2, 1, 8), state)
    with pytest.raises(ValueError, match="state must be float32"):
        ops.gated_step(x, x, state.half())
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        ops.gated_step(x, x, state)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        ops.gated_scan(_x(2, 4, 8), _x(2, 4, 8))


def _scan_args(batch=2, length=300, width=64, dtype=_hip.BF16, gate=True):
    """Fake, aligned device pointers: only host checks run on them."""
    args = _hip.GatedScanArgs(batch=batch, length=length, width=width, dtype=dtype)
    for i, name in enumerate(("x", "decay", "gate", "out")):
        if name == "gate" and not gate:
            continue
        t = getattr(args, name)
        t.ptr, t.dtype = 0x100000 * (i + 1), dtype
        t.stride[0], t.stride[1], t.stride[2] = length * width, width, 1
    if gate:
        args.rate = _hip.Tensor(0x600000, _hip.F32, 0, (1,))
    args.final_state = _hip.Tensor(0x700000, _hip.F32, 0, (width, 1))
    return args


def test_scan_validation_on_the_host(lib):
    size = ctypes.c_size_t(0)
    query = lib.m3_gated_scan_workspace_size
    assert query(ctypes.byref(_scan_args()), ctypes.byref(size)) == 0
    assert query(None, ctypes.byref(size)) == 1 and b"NULL" in lib.m3_last_error()
    assert lib.m3_gated_scan(None, None) == 1 and lib.m3_gated_scan_bwd(None, None) == 1
    for field, value, code, text in (("batch", -1, 1, b"negative"), ("dtype", 7, 1, b"dtype 7"),
                                     ("batch", 1 << 25, 2, b"above 2^30"),
                                     ("width", 1 << 28, 2, b"above 2^27")):
        args = _scan_args()
        setattr(args, field, value)
        assert query(ctypes.byref(args), ctypes.byref(size)) == code, field
        assert text in lib.m3_last_error()
    args = _scan_args()
    args.gate.ptr = None
    assert query(ctypes.byref(args), ctypes.byref(size)) == 1 and b"together" in lib.m3_last_error()
    args = _scan_args()
    args.x.stride[2] = 2
    assert query(ctypes.byref(args), ctypes.byref(size)) == 2
    args = _scan_args()
    args.decay.dtype = _hip.F32
    assert query(ctypes.byref(args), ctypes.byref(size)) == 2 and b"decay" in lib.m3_last_error()
    args = _scan_args()
    args.carry = _hip.Tensor(0x800000, _hip.F32, 0, (64, 64, 1))
    assert query(ctypes.byref(args), ctypes.byref(size)) == 2 and b"carry" in lib.m3_last_error()
    args = _scan_args(batch=0)
    assert lib.m3_gated_scan(ctypes.byref(args), None) == 0  # nothing to do


def test_backward_validation_on_the_host(lib):
    size = ctypes.c_size_t(0)

    def bwd():
        args = _hip.GatedScanBwdArgs(_scan_args())
        for i, name in enumerate(("dout", "dx", "ddecay", "dgate")):
            t = getattr(args, name)
            t.ptr, t.dtype = 0x1000000 * (i + 1), _hip.BF16
            t.stride[0], t.stride[1], t.stride[2] = 300 * 64, 64, 1
        args.drate = _hip.Tensor(0x900000, _hip.F32, 0, (1,))
        args.fwd.carry = _hip.Tensor(0xa00000, _hip.F32, 0, (2 * 64, 64, 1))
        return args

    query = lib.m3_gated_scan_bwd_workspace_size
    assert query(ctypes.byref(bwd()), ctypes.byref(size)) == 0 and size.value > 0
    assert lib.m3_gated_scan_bwd(ctypes.byref(bwd()), None) == 4  # no workspace
    assert b"workspace" in lib.m3_last_error()
    args = bwd()
    args.fwd.carry.ptr = None
    assert query(ctypes.byref(args), ctypes.byref(size)) == 1 and b"carry" in lib.m3_last_error()
    args = bwd()
    args.drate.ptr = None
    assert query(ctypes.byref(args), ctypes.byref(size)) == 1 and b"drate" in lib.m3_last_error()


def test_packed_blocks_put_every_value_in_its_field():
    """A block packed from 1, 2, 3, ... reads back so, field by field, through the structure."""
    def flat(value):
        if isinstance(value, ctypes.Structure):
            for name, _ in value._fields_:
                yield from flat(getattr(value, name))
        elif isinstance(value, ctypes.Array):
            yield from value
        else:
            yield value

    for packed, py in ((_hip.GATED_SCAN, _hip.GatedScanArgs),
                       (_hip.GATED_SCAN_BWD, _hip.GatedScanBwdArgs),
                       (_hip.LINEAR4, _hip.Linear4Args)):
        count = len(list(flat(py())))
        assert packed.size == ctypes.sizeof(py)
        read = py.from_buffer_copy(packed.pack(*range(1, count + 1)))
        assert list(flat(read)) == list(range(1, count + 1))


def test_structs_match_the_header_layout(tmp_path):
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {"m3_gated_scan_args": _hip.GatedScanArgs,
               "m3_gated_scan_bwd_args": _hip.GatedScanBwdArgs}
    for packed, py in ((_hip.GATED_SCAN, _hip.GatedScanArgs),
                       (_hip.GATED_SCAN_BWD, _hip.GatedScanBwdArgs)):
        assert packed.size == ctypes.sizeof(py)
    lines = ['#include "mamba3_hip.h"', "#include <stdio.h>", "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} - %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    lines.append(f'printf("tile - %d\\n", M3_GATED_TILE); return 0; }}')
    source = tmp_path / "layout.c"
    source.write_text("\n".join(lines))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{os.path.join(ROOT, 'include')}", str(source), "-o",
                    str(tmp_path / "layout")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True)
    for line in out.stdout.splitlines():
        cname, field, value = line.split()
        if cname == "tile":
            assert int(value) == _hip.GATED_TILE
        elif field == "-":
            assert ctypes.sizeof(structs[cname]) == int(value)
        else:
            assert getattr(structs[cname], field).offset == int(value), (cname, field)


def test_forward_mode_derivatives_are_refused():
    """Not dropped: a dual tensor has no requires_grad."""
    import torch.autograd.forward_ad as fwd
    x, weight = _x(2, 8), _x(8)
    with fwd.dual_level():
        for at in range(4):
            case = [_x(2, 4, 8), _x(2, 4, 8), _x(2, 4, 8), weight]
            case[at] = fwd.make_dual(case[at], torch.ones_like(case[at]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.gated_scan(*case)
        dual = fwd.make_dual(x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.gated_scan(_x(2, 4, 8), _x(2, 4, 8), initial_state=dual)
        with torch.no_grad():
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.gated_step(x, x, dual)
            held = ops.Weight4(torch.zeros(4, 16, dtype=torch.uint8), _x(4, 1, dtype=torch.float16))
            row = torch.zeros(1, 32, dtype=torch.float16)
            with pytest.raises(RuntimeError, match="forward-mode"):
                ops.linear4(fwd.make_dual(row, row), held)
            with pytest.raises(RuntimeError, match="ROCm devices only"):
                ops.linear4(row, held)  # a tensor without a tangent is none of its business


@pytest.mark.parametrize("length", [(1 << 30) + 1, (1 << 31) - 127, (1 << 31) - 1])
def test_a_length_beyond_the_tiles_of_a_grid(lib, length):
    """Refused as such: rounding it up to whole tiles would leave 32 bits."""
    size = ctypes.c_size_t(0)
    args = _scan_args(batch=1, width=1)
    args.length = length
    assert lib.m3_gated_scan_workspace_size(ctypes.byref(args), ctypes.byref(size)) == 2
    assert b"2^30" in lib.m3_last_error()
    assert lib.m3_gated_scan(ctypes.byref(args), None) == 2
    back = _hip.GatedScanBwdArgs(args)
    assert lib.m3_gated_scan_bwd_workspace_size(ctypes.byref(back), ctypes.byref(size)) == 2
    assert b"2^30" in lib.m3_last_error()
