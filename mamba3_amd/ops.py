"""Mamba-3 hot-path operators, executed by the HIP library (``include/mamba3_hip.h``).

Mirrors the operator interface of the reference ``mamba3/ops.py`` (jreoka/mamba3): the
same function names, argument meanings and ``ValueError`` validation messages. The
difference is the dispatch contract: the reference's hooks (``fused_step``,
``_fused_chunk_scan``) return ``None`` to fall back to a portable PyTorch path. This
package has no fallback. Every call runs the HIP kernels on a ROCm device or raises:
``RuntimeError`` for CPU tensors, for autograd use, and for a missing library;
``HipError`` for a failing call.

Module flags ``_HIP_LAST_DISPATCH`` / ``_HIP_LAST_SCAN_DISPATCH`` record that the last
step / scan ran on the HIP path (the reference's ``_TRITON_LAST_DISPATCH`` /
``_TRITON_LAST_SCAN_DISPATCH``, ``ops.py:14,18``).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _hip

_HIP_LAST_DISPATCH = False
_HIP_LAST_SCAN_DISPATCH = False
NORM_EPS = 1e-5
# Sequence segments of a scan call: 0 lets the library split long sequences of few (batch,
# head) pairs over more workgroups (two passes and a composition of the segment states); 1 never
# splits; G > 1 asks for G equal segments.
SCAN_SEGMENTS = 0


def heavy_tail_activation(x: torch.Tensor) -> torch.Tensor:
    """``1 + x`` for ``x >= 0``, ``1 / (1 - x)`` otherwise (reference ``ops.py:28-32``).

    Kept under the reference's name for callers that import it; no path of this package
    calls it: the kernels apply the activation to the raw ``dd_A`` logits themselves.
    """
    return torch.where(x >= 0, 1.0 + x, torch.reciprocal(1.0 - x.clamp_max(0)))


def _require_device(*tensors: torch.Tensor | None) -> torch.device:
    device = None
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError(
                "mamba3_amd runs the Mamba-3 hot path on ROCm devices only "
                f"(got a tensor on {t.device}); there is no CPU path")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RuntimeError("all tensors must be on the same device")
    if device is None:
        raise RuntimeError("no device tensor given")
    return device


def _require_inference(*tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in tensors]):
        raise RuntimeError(
            "mamba3_amd implements the inference hot path (forward, prefill, step) and has no "
            "backward; run it under torch.no_grad() or torch.inference_mode()")


def _refuse_tangents(*tensors: torch.Tensor | None) -> None:
    """Forward-mode derivatives, which need no ``requires_grad`` and outlast ``no_grad``, are refused
    where they would be dropped (call it only inside a dual level)."""
    if any([t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors]):
        raise RuntimeError("mamba3_amd has no forward-mode derivatives")


def _written(t: torch.Tensor) -> None:
    """Count a kernel's write into a caller's tensor, so that a backward pass that saved it (a
    ``gated_scan``'s) is refused instead of reading the new values."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _inner(t: torch.Tensor | None) -> torch.Tensor | None:
    """A view whose innermost axis has stride 1 (copy only when it does not)."""
    if t is None or t.dim() == 0 or t.shape[-1] <= 1 or t.stride(-1) == 1:
        return t
    return t.contiguous()


def _state32(t: torch.Tensor) -> torch.Tensor:
    t = t if t.dtype == torch.float32 else t.float()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 4 for s in t.stride()[:-1]):
        t = t.contiguous()
    return t


def _param(t: torch.Tensor | None) -> torch.Tensor | None:
    """Small parameter tensors: contiguous, any of f32 / bf16 / f16."""
    if t is None:
        return None
    t = t.detach()
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        t = t.float()
    return t.contiguous()


# --------------------------------------------------------------------------- scan


def _validate_scan(q, k, value, gate, adt, dt, trap_logits, D, mimo_x, mimo_z, mimo_out,
                   chunk_size, initial_state, initial_k, initial_value, phase, q_bias, k_bias):
    """Argument checks of the reference ``mamba3_scan`` (``ops.py:574-631``)."""
    if q.shape != k.shape or q.ndim != 5:
        raise ValueError("q and k must have matching [B, L, G, R, N] shapes")
    batch, length, qk_heads, rank, d_state = q.shape
    if value.ndim != 4 or gate.shape != value.shape:
        raise ValueError("value and gate must have matching [B, L, H, P] shapes")
    if value.shape[:2] != (batch, length):
        raise ValueError("value dimensions must match q and k")
    heads = value.shape[2]
    if heads % qk_heads != 0:
        raise ValueError("value heads must be divisible by Q/K groups")
    if adt.shape != (batch, length, heads):
        raise ValueError("adt must have shape [B, L, H]")
    if dt.shape != adt.shape or trap_logits.shape != adt.shape:
        raise ValueError("dt and trap_logits must match adt")
    if D.shape != (heads,):
        raise ValueError("D must have shape [H]")
    if (q_bias is None) != (k_bias is None):
        raise ValueError("q_bias and k_bias must be provided together")
    if q_bias is not None:
        expected_bias = (heads, rank, d_state)
        if q_bias.shape != expected_bias or k_bias.shape != expected_bias:
            raise ValueError(f"Q/K biases must have shape {expected_bias}")
    if chunk_size <= 0:
        raise ValueError("chunk_size must be positive")
    if phase is not None and (phase.ndim != 4 or phase.shape[:3] != (batch, length, heads)):
        raise ValueError("phase must have shape [B, L, H, S]")
    head_dim = value.shape[-1]
    expected_state = (batch, heads, head_dim, d_state)
    if initial_state is not None and initial_state.shape != expected_state:
        raise ValueError(f"initial_state must have shape {expected_state}")
    projections = (mimo_x, mimo_z, mimo_out)
    if rank == 1:
        if any(p is not None for p in projections):
            raise ValueError("SISO inputs must not provide MIMO projections")
    else:
        expected_projection = (heads, rank, head_dim)
        if any(p is None or p.shape != expected_projection for p in projections):
            raise ValueError(f"MIMO projections must have shape {expected_projection}")
    if initial_k is not None or initial_value is not None:
        expected_k = (batch, heads, rank, d_state)
        expected_value = (batch, heads, head_dim)
        if initial_k is None or initial_k.shape != expected_k:
            raise ValueError(f"initial_k must have shape {expected_k}")
        if initial_value is None or initial_value.shape != expected_value:
            raise ValueError(f"initial_value must have shape {expected_value}")


def mamba3_scan(q, k, value, gate, adt, dt, trap_logits, D, *, mimo_x=None, mimo_z=None,
                mimo_out=None, chunk_size=64, initial_state=None, initial_k=None,
                initial_value=None, phase=None, mimo_rotation=False, q_bias=None, k_bias=None):
    """Chunked Mamba-3 SSD with an FP32 state (reference ``ops.py:544-822``).

    ``q/k [B,L,G,R,N]`` (RMS-normed, unbiased, unrotated), ``value/gate [B,L,H,P]``,
    ``adt/dt [B,L,H]`` FP32, ``trap_logits [B,L,H]``, optional ``phase [B,L,H,S]`` FP32.
    Returns ``(output [B,L,H,P], state [B,H,P,N] FP32)``. One HIP launch for the whole
    sequence; ``chunk_size`` is validated and passed on as advisory.
    """
    global _HIP_LAST_SCAN_DISPATCH
    _HIP_LAST_SCAN_DISPATCH = False
    _validate_scan(q, k, value, gate, adt, dt, trap_logits, D, mimo_x, mimo_z, mimo_out,
                   chunk_size, initial_state, initial_k, initial_value, phase, q_bias, k_bias)
    device = _require_device(q, k, value, gate, adt, dt, trap_logits, D, initial_state,
                             initial_k, initial_value, phase, q_bias, k_bias, mimo_x)
    _require_inference(q, k, value, gate, adt, dt, trap_logits, D, mimo_x, mimo_z, mimo_out,
                       initial_state, initial_k, initial_value, phase, q_bias, k_bias)
    batch, length, groups, rank, d_state = q.shape
    heads, head_dim = value.shape[2], value.shape[3]
    if not (q.dtype == k.dtype == value.dtype == gate.dtype):
        raise ValueError("q, k, value and gate must share one dtype")
    state_in = None if initial_state is None else _state32(initial_state)
    final_state = torch.empty(batch, heads, head_dim, d_state, device=device,
                              dtype=torch.float32)
    if length == 0 or batch == 0:
        if state_in is None:
            final_state.zero_()
        else:
            final_state.copy_(state_in)
        return value.clone(), final_state
    out = torch.empty(batch, length, heads, head_dim, device=device, dtype=value.dtype)
    num_angles = 0 if phase is None else phase.shape[-1]
    args = _hip.ScanArgs(
        batch=batch, length=length, heads=heads, groups=groups, rank=rank, d_state=d_state,
        head_dim=head_dim, num_angles=num_angles, chunk=chunk_size,
        act_dtype=_hip.dtype_code(q.dtype), mimo_rotation=int(bool(mimo_rotation)), raw_dt=0,
        phase_mode=_hip.PHASE_NONE if phase is None else _hip.PHASE_GIVEN, norm_eps=NORM_EPS,
        segments=SCAN_SEGMENTS)
    keep = [_inner(q), _inner(k), _inner(value), _inner(gate), adt.float(), dt.float(),
            trap_logits, None if phase is None else phase.float(), _param(D), _param(mimo_x),
            _param(mimo_z), _param(mimo_out), _param(q_bias), _param(k_bias), state_in,
            _inner(initial_k), _inner(initial_value)]
    (args.q, args.k, args.value, args.gate, args.a, args.dt, args.trap, args.phase, args.D,
     args.mimo_x, args.mimo_z, args.mimo_out, args.q_bias, args.k_bias, args.initial_state,
     args.initial_k, args.initial_value) = (_hip.tensor(t) for t in keep)
    args.out = _hip.tensor(out)
    args.final_state = _hip.tensor(final_state)
    with torch.cuda.device(device):
        keep.append(_hip.scan_workspace(args, device))
        _hip.call("m3_scan_fwd", args, device)
    _HIP_LAST_SCAN_DISPATCH = True
    return out, final_state


def chunk_state(k, value, cumulative, scale, state, output, *, width: int, rank: int) -> None:
    """One chunk's state update (reference ``_triton.py:500-561``), written into ``output``.

    ``k [B,H,W,R,N]`` biased and rotated, ``value [B,H,W,R,P]`` rank values,
    ``cumulative/scale [B,H,W]`` FP32, ``state/output [B,H,P,N]`` FP32 (may be the same).
    """
    device = _require_device(k, value, cumulative, scale, state, output)
    batch, heads, head_dim, d_state = state.shape
    if k.shape[2] < width or value.shape[2] < width:
        raise ValueError("width exceeds the chunk tensors")
    if output.dtype != torch.float32 or state.dtype != torch.float32:
        raise ValueError("state and output must be float32")
    args = _hip.ChunkStateArgs(batch=batch, width=width, heads=heads, rank=rank,
                               d_state=d_state, head_dim=head_dim,
                               act_dtype=_hip.dtype_code(k.dtype))
    keep = [_inner(k), _inner(value), cumulative.float(), scale.float(), _inner(state)]
    args.k, args.value, args.cumulative, args.scale, args.state_in = (
        _hip.tensor(t) for t in keep)
    if output.stride(-1) != 1:
        raise ValueError("output must have a unit innermost stride")
    args.state_out = _hip.tensor(output)
    with torch.cuda.device(device):
        _hip.call("m3_chunk_state", args, device)


# --------------------------------------------------------------------------- step


def _step_call(q, k, value, gate, adt, dt, trap_logits, angle_rate, D, cache, *, mimo_x,
               mimo_z, mimo_out, phase_mode, raw=None, out_cache=None):
    phase, state, prev_k, prev_v = cache
    device = _require_device(q, k, value, gate, state, prev_k, prev_v, D)
    batch, groups, rank, d_state = q.shape
    heads, head_dim = value.shape[1], value.shape[2]
    num_angles = phase.shape[-1]
    out = torch.empty(batch, heads, head_dim, device=device, dtype=value.dtype)
    if out_cache is None:
        phase_out = torch.empty(batch, heads, num_angles, device=device, dtype=torch.float32)
        state_out = torch.empty(batch, heads, head_dim, d_state, device=device,
                                dtype=torch.float32)
        k_out = torch.empty(batch, heads, rank, d_state, device=device, dtype=q.dtype)
        value_out = None
    else:
        phase_out, state_out, k_out, value_out = out_cache
    if batch == 0:
        return out, (phase_out, state_out, k_out, value if value_out is None else value_out)
    args = _hip.StepArgs(batch=batch, heads=heads, groups=groups, rank=rank, d_state=d_state,
                         head_dim=head_dim, num_angles=num_angles,
                         act_dtype=_hip.dtype_code(q.dtype), mimo_rotation=int(rank > 1),
                         raw_dt=int(raw is not None), phase_mode=phase_mode, norm_eps=NORM_EPS)
    keep = [_inner(q), _inner(k), _inner(value), _inner(gate), dt, adt, trap_logits,
            angle_rate, _param(D), _param(mimo_x), _param(mimo_z), _param(mimo_out),
            phase, _state32(state), _inner(prev_k), _inner(prev_v)]
    (args.q, args.k, args.value, args.gate, args.dt, args.a, args.trap, args.angles, args.D,
     args.mimo_x, args.mimo_z, args.mimo_out, args.phase_in, args.state_in, args.prev_k,
     args.prev_value) = (_hip.tensor(t) for t in keep)
    if raw is not None:
        q_norm_w, k_norm_w, q_bias, k_bias, dt_bias = (_param(t) for t in raw)
        keep += [q_norm_w, k_norm_w, q_bias, k_bias, dt_bias]
        args.q_norm_w, args.k_norm_w = _hip.tensor(q_norm_w), _hip.tensor(k_norm_w)
        args.q_bias, args.k_bias = _hip.tensor(q_bias), _hip.tensor(k_bias)
        args.dt_bias = _hip.tensor(dt_bias)
    args.out = _hip.tensor(out)
    args.phase_out = _hip.tensor(phase_out)
    args.state_out = _hip.tensor(state_out)
    args.k_out = _hip.tensor(k_out)
    args.value_out = _hip.tensor(value_out)
    with torch.cuda.device(device):
        _hip.call("m3_step", args, device)
    return out, (phase_out, state_out, k_out, value if value_out is None else value_out)


def _validate_step_shapes(q, k, value, gate, adt, dt, trap_logits, D, cache, mimo_x, mimo_z,
                          mimo_out, angle_rate=None):
    """Shape checks of the reference fused step launcher (``_triton.py:968-1044``)."""
    phase, state, previous_k, previous_value = cache
    if q.ndim != 4 or q.shape != k.shape:
        raise ValueError("q and k must have the same [B, H, R, N] shape")
    batch, heads, rank, d_state = q.shape
    head_dim = value.shape[-1]
    num_angles = phase.shape[-1]
    expected = {
        "value": (batch, heads, head_dim), "gate": (batch, heads, head_dim),
        "adt": (batch, heads), "dt": (batch, heads), "trap_logits": (batch, heads),
        "D": (heads,), "phase": (batch, heads, num_angles),
        "state": (batch, heads, head_dim, d_state),
        "previous_k": (batch, heads, rank, d_state),
        "previous_value": (batch, heads, head_dim),
    }
    given = {"value": value, "gate": gate, "adt": adt, "dt": dt, "trap_logits": trap_logits,
             "D": D, "phase": phase, "state": state, "previous_k": previous_k,
             "previous_value": previous_value}
    if angle_rate is not None:
        expected["angle_rate"] = (batch, num_angles)
        given["angle_rate"] = angle_rate
    for name, shape in expected.items():
        if tuple(given[name].shape) != shape:
            raise ValueError(f"invalid {name} shape: expected {shape}, "
                             f"got {tuple(given[name].shape)}")
    if not (q.dtype == k.dtype == value.dtype == gate.dtype):
        raise ValueError("q, k, value, and gate must have the same dtype")
    if previous_k.dtype != q.dtype or previous_value.dtype != value.dtype:
        raise ValueError("K/value cache dtypes must match current activations")
    if phase.dtype != torch.float32 or state.dtype != torch.float32:
        raise ValueError("phase and state must be float32")
    if rank > 1:
        for name, proj in (("mimo_x", mimo_x), ("mimo_z", mimo_z), ("mimo_out", mimo_out)):
            if proj is None or proj.shape != (heads, rank, head_dim):
                raise ValueError(f"invalid {name} shape: expected {(heads, rank, head_dim)}")
    elif mimo_x is not None:
        raise ValueError("MIMO projections require rank > 1")


def fused_step(q, k, value, gate, adt, dt, trap_logits, angle_rate, D, cache, *, mimo_x=None,
               mimo_z=None, mimo_out=None):
    """One decode token with the phase advance and rotation fused (``ops.py:87-190``).

    Inputs are head-expanded, biased and unrotated: ``q/k [B,H,R,N]``, ``value/gate
    [B,H,P]``, ``adt/dt/trap_logits [B,H]``, ``angle_rate [B,S]``; ``cache = (phase
    [B,H,S] FP32, state [B,H,P,N] FP32, prev_k [B,H,R,N], prev_value [B,H,P])``.
    Returns ``(output [B,H,P], (phase', state', k_rot, value))``.
    """
    global _HIP_LAST_DISPATCH
    _HIP_LAST_DISPATCH = False
    _validate_step_shapes(q, k, value, gate, adt, dt, trap_logits, D, cache, mimo_x, mimo_z,
                          mimo_out, angle_rate)
    _require_inference(q, k, value, gate, adt, dt, trap_logits, angle_rate, D, *cache)
    result = _step_call(q, k, value, gate, adt, dt, trap_logits, angle_rate, D, cache,
                        mimo_x=mimo_x, mimo_z=mimo_z, mimo_out=mimo_out,
                        phase_mode=_hip.PHASE_ANGLES)
    _HIP_LAST_DISPATCH = True
    return result


def mamba3_step(q, k, value, gate, adt, dt, trap_logits, D, cache, *, mimo_x=None,
                mimo_z=None, mimo_out=None):
    """One exact recurrent update with rotated ``q/k [B,H,R,N]`` (``ops.py:825-879``).

    The cache phase is passed through unchanged.
    """
    global _HIP_LAST_DISPATCH
    _HIP_LAST_DISPATCH = False
    _validate_step_shapes(q, k, value, gate, adt, dt, trap_logits, D, cache, mimo_x, mimo_z,
                          mimo_out)
    _require_inference(q, k, value, gate, adt, dt, trap_logits, D, *cache)
    out, nxt = _step_call(q, k, value, gate, adt, dt, trap_logits, None, D, cache,
                          mimo_x=mimo_x, mimo_z=mimo_z, mimo_out=mimo_out,
                          phase_mode=_hip.PHASE_NONE)
    _HIP_LAST_DISPATCH = True
    return out, nxt


# --------------------------------------------------------------------------- projection form


def split_projection(proj: torch.Tensor, mixer) -> dict[str, torch.Tensor]:
    """Views into the ``in_proj`` output in the reference split order (``model.py:147-163``):
    ``[z, x, B, C, dd_dt, dd_A, trap, angles]``."""
    d_inner, n, r = mixer.d_inner, mixer.d_state, mixer.mimo_rank
    h, p, s = mixer.nheads, mixer.headdim, mixer.num_angles
    sizes = (d_inner, d_inner, n * r, n * r, h, h, h, s)
    z, x, b, c, ddt, da, trap, ang = torch.split(proj, sizes, dim=-1)
    lead = proj.shape[:-1]
    return dict(
        z=z.unflatten(-1, (h, p)), x=x.unflatten(-1, (h, p)),
        k=b.unflatten(-1, (1, r, n)), q=c.unflatten(-1, (1, r, n)),
        dt=ddt, a=da, trap=trap, angles=ang, lead=lead)


def _backwards(desc: _hip.Tensor, length: int) -> None:
    """Make a per-token descriptor run backwards: token t at the old token L - 1 - t."""
    if desc.ptr is None or length <= 1:
        return
    size = 4 if desc.dtype == _hip.F32 else 2
    desc.ptr += (length - 1) * desc.stride[1] * size
    desc.stride[1] = -desc.stride[1]


class ScanCall:
    """One ``m3_scan_fwd`` launch over the raw ``in_proj`` output ``[B, L, proj]``, prepared once.

    Holds the argument block, the outputs, the workspace and references to every tensor the
    block points at; ``launch()`` enqueues the call on the device's current stream and may be
    repeated (each launch rewrites the outputs). Fuses the reference mixer's ``_project`` (B/C
    RMSNorm, dt, adt; ``model.py:165``), ``_phase`` (``model.py:215``), bias, rotation and the
    chunked SSD (reference ``model.py:282-309``).

    ``reverse=True`` scans the sequence from its last token to its first, reading ``proj`` and
    writing ``out`` through backwards token strides: ``out`` then holds, in forward order,
    what scanning ``flip(proj)`` and flipping the result back gives (the reverse direction of
    a bidirectional layer, reference ``model.py:330-362``, without either flip or a second
    projection).

    ``concurrent``: how many calls of this shape run at once (2 for the two directions of a
    bidirectional layer). A long sequence of few (batch, head) pairs is split into segments
    sized for the calls' combined grid, unless ``SCAN_SEGMENTS`` fixes the split.
    """

    def __init__(self, proj: torch.Tensor, mixer, *, cache=None, want_cache: bool = False,
                 chunk_size: int = 256, reverse: bool = False, concurrent: int = 1):
        self.device = _require_device(proj)
        v = split_projection(proj, mixer)
        batch, length = proj.shape[0], proj.shape[1]
        h, p, n, r = mixer.nheads, mixer.headdim, mixer.d_state, mixer.mimo_rank
        s = mixer.num_angles
        act = proj.dtype
        if cache is not None:
            init_phase, init_state, init_k, init_v = cache
            if init_k.dtype != act or init_v.dtype != act:
                raise ValueError("K/value cache dtypes must match the activations")
        else:
            init_phase = init_state = init_k = init_v = None
        dev = self.device
        self.out = torch.empty(batch, length, h, p, device=dev, dtype=act)
        self.final_state = torch.empty(batch, h, p, n, device=dev, dtype=torch.float32)
        self.final_phase = (torch.empty(batch, h, s, device=dev, dtype=torch.float32)
                            if want_cache else None)
        self.final_k = torch.empty(batch, h, r, n, device=dev, dtype=act) if want_cache else None
        args = _hip.ScanArgs(
            batch=batch, length=length, heads=h, groups=1, rank=r, d_state=n, head_dim=p,
            num_angles=s, chunk=chunk_size, act_dtype=_hip.dtype_code(act),
            mimo_rotation=int(r > 1), raw_dt=1, phase_mode=_hip.PHASE_ANGLES,
            norm_eps=NORM_EPS, segments=SCAN_SEGMENTS)
        params = [_param(t) for t in (mixer.C_norm.weight, mixer.B_norm.weight, mixer.C_bias,
                                      mixer.B_bias, mixer.dt_bias, mixer.D, mixer.mimo_x,
                                      mixer.mimo_z, mixer.mimo_out)]
        keep = [v["q"], v["k"], v["x"], v["z"], v["dt"], v["a"], v["trap"], v["angles"],
                init_phase, None if init_state is None else _state32(init_state),
                _inner(init_k), _inner(init_v), *params]
        (args.q, args.k, args.value, args.gate, args.dt, args.a, args.trap, args.phase,
         args.initial_phase, args.initial_state, args.initial_k, args.initial_value,
         args.q_norm_w, args.k_norm_w, args.q_bias, args.k_bias, args.dt_bias, args.D,
         args.mimo_x, args.mimo_z, args.mimo_out) = (_hip.tensor(t) for t in keep)
        args.out = _hip.tensor(self.out)
        args.final_state = _hip.tensor(self.final_state)
        args.final_phase = _hip.tensor(self.final_phase)
        args.final_k = _hip.tensor(self.final_k)
        if reverse:
            if cache is not None or want_cache:
                raise ValueError("a reverse scan has no cache")
            for desc in (args.q, args.k, args.value, args.gate, args.dt, args.a, args.trap,
                         args.phase, args.out):
                _backwards(desc, length)
        if concurrent > 1 and args.segments == 0:
            # `concurrent` calls of this shape share the GPU (the two directions of a
            # bidirectional layer): the library's segment choice for their combined grid
            args.segments = _hip.scan_segments(args, concurrent)
        with torch.cuda.device(dev):
            keep.append(_hip.scan_workspace(args, dev))
        self.args = args
        self._keep = keep

    def launch(self) -> None:
        global _HIP_LAST_SCAN_DISPATCH
        _HIP_LAST_SCAN_DISPATCH = False
        with torch.cuda.device(self.device):
            _hip.call("m3_scan_fwd", self.args, self.device)
        _HIP_LAST_SCAN_DISPATCH = True


def scan_projection(proj: torch.Tensor, mixer, *, cache=None, want_cache: bool = False,
                    chunk_size: int = 256, reverse: bool = False, concurrent: int = 1):
    """The whole mixer scan from the raw ``in_proj`` output ``[B, L, proj]``.

    Fuses the reference mixer's ``_project`` (B/C RMSNorm, dt, adt; ``model.py:165``),
    ``_phase``, bias, rotation and the chunked SSD (reference ``model.py:282-309``). Returns ``(mixed [B,L,H,P], state, final_phase,
    final_k)``; the last two are ``None`` unless ``want_cache``. ``reverse``, ``concurrent``: see
    ``ScanCall``.
    """
    call = ScanCall(proj, mixer, cache=cache, want_cache=want_cache, chunk_size=chunk_size,
                    reverse=reverse, concurrent=concurrent)
    call.launch()
    return call.out, call.final_state, call.final_phase, call.final_k


def step_projection(proj: torch.Tensor, mixer, cache, *, inplace: bool = False):
    """One decode token from the raw ``in_proj`` output ``[B, 1, proj]``.

    Fuses the reference mixer's ``_project`` and ``_expand_qk`` (``model.py:165``, ``201``),
    the phase advance, the rotation and the step (reference ``model.py:431-484``). With ``inplace`` the cache tensors are updated in
    place (the hipGraph decoder's static cache) and returned.
    """
    global _HIP_LAST_DISPATCH
    _HIP_LAST_DISPATCH = False
    v = split_projection(proj[:, 0], mixer)  # q, k: [B, G=1, R, N]; x, z: [B, H, P]
    q, k = v["q"], v["k"]
    out_cache = cache if inplace else None
    out, nxt = _step_call(
        q, k, v["x"], v["z"], v["a"], v["dt"], v["trap"], v["angles"], mixer.D, cache,
        mimo_x=mixer.mimo_x, mimo_z=mixer.mimo_z, mimo_out=mixer.mimo_out,
        phase_mode=_hip.PHASE_ANGLES,
        raw=(mixer.C_norm.weight, mixer.B_norm.weight, mixer.C_bias, mixer.B_bias,
             mixer.dt_bias),
        out_cache=out_cache)
    _HIP_LAST_DISPATCH = True
    return out, nxt


# --------------------------------------------------------------------------- decode GEMMs

LINEAR_MAX_ROWS = 256
# The fused RMSNorm takes up to 32 rows, or up to 64 when K is a multiple of 256.
LINEAR_NORM_MAX_ROWS = 64
# Decode steps run in_proj (with the block's RMSNorm fused) on ``linear`` up to
# DECODE_LINEAR_ROWS rows, and out_proj (with the residual add fused) up to
# DECODE_LINEAR_OUT_ROWS. Measured on the decode shapes with cold weights: above these, hipBLASLt
# (plus the separate norm or add) is faster.
DECODE_LINEAR_ROWS = 64
DECODE_LINEAR_OUT_ROWS = 64


def linear_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether ``linear(x, weight)`` takes these operands: 2-D, on one ROCm device, both
    bfloat16 or both float16, at most ``LINEAR_MAX_ROWS`` rows, K a multiple of 32 with
    16-byte aligned rows, no autograd, and no autocast that would compute in another dtype."""
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        return False
    if x.device.type != "cuda" or weight.device != x.device:
        return False
    if x.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != x.dtype:
        return False
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != x.dtype:
        return False
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return False
    m, k = x.shape
    if not 0 < m <= LINEAR_MAX_ROWS or k % 32 != 0 or weight.shape[0] == 0:
        return False
    for t in (x, weight):
        if t.stride(1) != 1 or t.stride(0) % 8 != 0 or t.data_ptr() % 16 != 0:
            return False
    return True


def linear_norm_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether ``linear(x, weight, norm_weight=...)`` takes these operands: ``linear_supported``
    and at most 32 rows, or at most ``LINEAR_NORM_MAX_ROWS`` with K a multiple of 256."""
    if not linear_supported(x, weight):
        return False
    m, k = x.shape
    return m <= 32 or (m <= LINEAR_NORM_MAX_ROWS and k % 256 == 0)


def linear(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
           out: torch.Tensor | None = None, norm_weight: torch.Tensor | None = None,
           norm_eps: float = NORM_EPS) -> torch.Tensor:
    """``x @ weight.T (+ residual)`` for the few rows of a decode step (``m3_linear``).

    ``x`` is ``[M, K]`` (``M <= 256``), ``weight`` the ``[N, K]`` weight of an ``nn.Linear``
    without bias, both bfloat16 or both float16 (``linear_supported``); ``residual`` and
    ``out`` are ``[M, N]`` of that dtype. Products accumulate in FP32; the residual is added
    to the FP32 sum, which is rounded once. With ``norm_weight`` (``[K]``; ``M <= 32``, or
    ``M <= 64`` with K a multiple of 256) ``x`` is first RMS-normalised, as
    ``F.rms_norm(x, (K,), norm_weight, norm_eps)``, with ``x * norm_weight`` rounded to ``x``'s
    dtype before the division (in float16 it has to stay below 65504). This replaces the decode
    step's RMSNorm, ``in_proj`` / ``out_proj`` calls and the block's residual add (reference
    ``model.py:441-458, 514-520``).
    """
    device = _require_device(x, weight, residual, out, norm_weight)
    _require_inference(x, weight, residual, norm_weight)
    if not linear_supported(x, weight):
        raise ValueError(
            f"linear: unsupported operands x {tuple(x.shape)} {x.dtype} strides {x.stride()}, "
            f"weight {tuple(weight.shape)} {weight.dtype} strides {weight.stride()}")
    m, n = x.shape[0], weight.shape[0]
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (tuple(t.shape) != (m, n) or t.dtype != x.dtype):
            raise ValueError(f"linear: {name} must be [{m}, {n}] {x.dtype}, got "
                             f"{tuple(t.shape)} {t.dtype}")
    if norm_weight is not None:
        if not linear_norm_supported(x, weight):
            raise ValueError(f"linear: norm_weight needs at most 32 rows, or at most "
                             f"{LINEAR_NORM_MAX_ROWS} with K a multiple of 256")
        norm_weight = norm_weight.detach().to(x.dtype).contiguous()
        if norm_weight.shape != (x.shape[1],):
            raise ValueError(f"linear: norm_weight must be [{x.shape[1]}]")
        if norm_weight.data_ptr() % 16:
            norm_weight = norm_weight.clone()
    residual, given = _inner(residual), out is not None
    if not given:
        out = torch.empty(m, n, dtype=x.dtype, device=device)
    elif out.stride(1) != 1:
        raise ValueError("linear: out needs a unit inner stride")
    args = _hip.LinearArgs()
    args.m, args.n, args.k = m, n, x.shape[1]
    args.dtype = _hip.dtype_code(x.dtype)
    args.x = _hip.tensor(x)
    args.weight = _hip.tensor(weight.detach())
    args.norm_weight = _hip.tensor(norm_weight)
    args.norm_eps = float(norm_eps)
    args.residual = _hip.tensor(residual)
    args.out = _hip.tensor(out)
    ws = _hip.scan_workspace(args, device, "m3_linear_workspace_size")
    _hip.call("m3_linear", args, device)
    del ws
    if given:
        _written(out)
    return out


# --------------------------------------------------------------------------- residual stream

RMS_NORM_DIMS = (256, 512, 768, 1024, 2048)
_FLOAT_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows_ok(t: torch.Tensor) -> bool:
    return t.is_contiguous() and t.data_ptr() % (4 * t.element_size()) == 0


def rms_norm_supported(x: torch.Tensor, weight: torch.Tensor, add: torch.Tensor | None = None,
                       out_dtype: torch.dtype | None = None) -> bool:
    """Whether ``rms_norm`` takes these operands: contiguous rows on one ROCm device, the last
    axis in ``RMS_NORM_DIMS``, an FP32 ``x`` with any ``add`` / ``out_dtype`` or a 16-bit ``x``
    with both of its own dtype, and no autograd."""
    out_dtype = out_dtype or x.dtype
    if x.device.type != "cuda" or x.dim() < 1 or x.shape[-1] not in RMS_NORM_DIMS:
        return False
    if x.dtype not in _FLOAT_DTYPES or out_dtype not in _FLOAT_DTYPES:
        return False
    if weight.device != x.device or tuple(weight.shape) != (x.shape[-1],):
        return False
    if weight.dtype not in _FLOAT_DTYPES or not _rows_ok(x):
        return False
    if add is not None:
        if add.device != x.device or add.shape != x.shape or not _rows_ok(add):
            return False
        if add.dtype not in _FLOAT_DTYPES or (x.dtype != torch.float32 and add.dtype != x.dtype):
            return False
    if x.dtype != torch.float32 and out_dtype != x.dtype:
        return False
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, add)):
        return False
    return True


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = NORM_EPS, *,
             add: torch.Tensor | None = None, keep_sum: bool = False,
             out_dtype: torch.dtype | None = None):
    """One pass of the residual stream (``m3_rms_norm``): ``s = x + add`` (or ``x``), then
    ``F.rms_norm(s, (d,), weight.to(s.dtype), eps)`` written as ``out_dtype`` (default
    ``x.dtype``). Returns ``(out, s)`` with ``s`` only when ``keep_sum`` (``add`` given).

    ``s`` is the reference's ``hidden_states + mixed`` (``model.py:511-512``; an FP32 ``x``
    takes an ``add`` of any dtype), ``out`` its next RMSNorm (``model.py:48-55``) already in
    the dtype the next projection computes in, so the add, the norm and autocast's cast are one
    pass over the rows instead of three.
    """
    out_dtype = out_dtype or x.dtype
    device = _require_device(x, weight, add)
    _require_inference(x, weight, add)
    if not rms_norm_supported(x, weight, add, out_dtype):
        raise ValueError(f"rms_norm: unsupported operands x {tuple(x.shape)} {x.dtype}, add "
                         f"{None if add is None else (tuple(add.shape), add.dtype)}, out "
                         f"{out_dtype}")
    if keep_sum and add is None:
        raise ValueError("rms_norm: keep_sum needs add")
    d = x.shape[-1]
    rows = x.numel() // d
    w = weight.detach()
    if w.data_ptr() % (4 * w.element_size()) or not w.is_contiguous():
        w = w.contiguous().clone()
    out = torch.empty(x.shape, dtype=out_dtype, device=device)
    s = torch.empty_like(x) if keep_sum else None
    if rows == 0:
        return out, s
    args = _hip.RmsNormArgs()
    args.rows, args.dim, args.eps = rows, d, float(eps)
    args.x = _hip.tensor(x.view(rows, d))
    args.add = _hip.tensor(None if add is None else add.view(rows, d))
    args.weight = _hip.tensor(w)
    args.sum_out = _hip.tensor(None if s is None else s.view(rows, d))
    args.out = _hip.tensor(out.view(rows, d))
    _hip.call("m3_rms_norm", args, device)
    return out, s


# --------------------------------------------------------------------------- 4-bit weights

LINEAR4_GROUPS = (32, 64, 128)


class Weight4:
    """An ``nn.Linear`` weight ``[N, K]`` held in 4 bits, laid out for ``linear4``.

    ``packed [N, K / 2]`` uint8: codes 0..15, the even column in the low four bits. ``scales [N,
    K / group]`` bfloat16 or float16, ``group`` 32, 64 or 128 by its shape; ``zeros`` of the same
    shape, uint8 0..15, or ``None`` for 8 everywhere. The weight is ``(code - zero) * scale``.
    The three are copied into the kernel's tiles once, here (``m3_linear4``'s layout: a wave reads
    a tile of 16 rows by 128 columns as 1 KB); later changes to them are not seen.
    """

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor,
                 zeros: torch.Tensor | None = None) -> None:
        if packed.ndim != 2 or packed.dtype != torch.uint8 or packed.numel() == 0:
            raise ValueError("packed must be uint8 of shape [N, K / 2]")
        n, k = packed.shape[0], 2 * packed.shape[1]
        if scales.ndim != 2 or scales.shape[0] != n or scales.numel() == 0:
            raise ValueError("scales must have shape [N, K / group]")
        if scales.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("scales must be bfloat16 or float16")
        group = k // scales.shape[1]
        if group not in LINEAR4_GROUPS or group * scales.shape[1] != k:
            raise ValueError(f"{scales.shape[1]} scales a row of {k}: groups must be of 32, 64 or 128")
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != torch.uint8):
            raise ValueError("zeros must be uint8 of the scales' shape")
        if any(t is not None and t.device != packed.device for t in (scales, zeros)):
            raise ValueError("packed, scales and zeros must be on the same device")
        if zeros is not None and bool((zeros > 15).any()):
            raise ValueError("zeros must be codes, 0 to 15")
        self.shape, self.group, self.device = (n, k), group, packed.device
        self.dtype = scales.dtype
        tn, tk = -(-n // 16), -(-k // 128)
        # [N, K] codes -> [tn, row, tk, word i, lane group, e] -> [tn, tk, lane group, row, i, e]
        codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(1)
        codes = torch.nn.functional.pad(codes, (0, 128 * tk - k, 0, 16 * tn - n))
        codes = codes.view(tn, 16, tk, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5)
        # a word's nibbles: the even columns, then the odd ones; two to a byte
        codes = codes.reshape(tn, tk, 64, 4, 8)
        self.codes = (codes[..., 0::2] | codes[..., 1::2] << 4).contiguous()
        self.scales = self._tiles(scales, tn, tk)
        self.zeros = None if zeros is None else self._tiles(zeros, tn, tk)

    def _tiles(self, t: torch.Tensor, tn: int, tk: int) -> torch.Tensor:
        per = 128 // self.group
        t = torch.nn.functional.pad(t.detach(), (0, per * tk - t.shape[1], 0, 16 * tn - t.shape[0]))
        return t.view(tn, 16, tk, per).permute(0, 2, 3, 1).contiguous()

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The weight ``[N, K]`` as ``(code - zero) * scale``, one product in FP32 rounded to
        ``dtype`` (default: the scales')."""
        n, k = self.shape
        tn, tk = self.codes.shape[:2]
        codes = torch.stack([self.codes & 15, self.codes >> 4], dim=-1)
        codes = codes.view(tn, tk, 4, 16, 4, 2, 4).permute(0, 3, 1, 4, 2, 6, 5)
        codes = codes.reshape(16 * tn, -1, self.group).float()

        def rows(t):
            return t.permute(0, 3, 1, 2).reshape(16 * tn, -1, 1).float()

        zeros = 8.0 if self.zeros is None else rows(self.zeros)
        weight = ((codes - zeros) * rows(self.scales)).flatten(1)
        return weight[:n, :k].to(dtype or self.dtype).contiguous()


def quantize4(weight: torch.Tensor, group: int = 128, *, zeros: bool = True,
              dtype: torch.dtype | None = None) -> Weight4:
    """``weight [N, K]`` rounded to 4 bits in groups of ``group`` columns.

    With ``zeros`` a group's codes span its least to its greatest value (0 among them, which stays
    exact); without, they are centred on code 8. Scales are ``dtype`` (default: the weight's, or
    bfloat16 for an FP32 weight), and codes are rounded with the scale as it is held.
    """
    if weight.ndim != 2 or weight.dtype not in _FLOAT_DTYPES or weight.numel() == 0:
        raise ValueError("weight must be a floating [N, K] tensor")
    if group not in LINEAR4_GROUPS or weight.shape[1] % group != 0:
        raise ValueError(f"quantize4: K = {weight.shape[1]} must be a multiple of group "
                         f"{group}, one of {LINEAR4_GROUPS}")
    dtype = dtype or (torch.bfloat16 if weight.dtype == torch.float32 else weight.dtype)
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("scales must be bfloat16 or float16")
    w = weight.detach().float().unflatten(1, (-1, group))
    if not bool(torch.isfinite(w).all()):
        raise ValueError("quantize4: the weight holds NaN or infinities")
    if zeros:
        low, high = w.amin(-1, keepdim=True).clamp(max=0), w.amax(-1, keepdim=True).clamp(min=0)
        scale = (high - low) / 15
    else:
        scale = torch.maximum(w.amax(-1, keepdim=True) / 7, -w.amin(-1, keepdim=True) / 8)
    scale = scale.to(dtype).float()
    if not bool(torch.isfinite(scale).all()):
        raise ValueError(f"quantize4: a group's range is beyond {dtype}")
    step = torch.where(scale > 0, scale, 1.0)
    zero = (-low / step).round().clamp(0, 15) if zeros else torch.full_like(scale, 8.0)
    codes = ((w / step).round() + zero).clamp(0, 15).to(torch.uint8).flatten(1)
    return Weight4(codes[:, 0::2] | codes[:, 1::2] << 4, scale.squeeze(-1).to(dtype),
                   zero.squeeze(-1).to(torch.uint8) if zeros else None)


def linear4_supported(x: torch.Tensor, weight: Weight4) -> bool:
    """Whether ``linear4(x, weight)`` takes these operands: 1 to ``LINEAR_MAX_ROWS`` rows of K
    bfloat16 or float16 values on the weight's ROCm device, no autograd, and no autocast that would
    compute in another dtype."""
    return (x.dim() == 2 and x.shape[1] == weight.shape[1] and 0 < x.shape[0] <= LINEAR_MAX_ROWS
            and x.device.type == "cuda" and x.device == weight.device
            and x.dtype in (torch.bfloat16, torch.float16)
            and not (torch.is_autocast_enabled("cuda")
                     and torch.get_autocast_dtype("cuda") != x.dtype)
            and not (torch.is_grad_enabled() and x.requires_grad))


def _aligned16(t: torch.Tensor) -> torch.Tensor:
    """``t`` with 16-byte aligned rows of unit inner stride (itself if it has them)."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and (t.dim() == 1 or t.stride(0) % 8 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def linear4(x: torch.Tensor, weight: Weight4, residual: torch.Tensor | None = None, *,
            out: torch.Tensor | None = None, norm_weight: torch.Tensor | None = None,
            norm_eps: float = NORM_EPS) -> torch.Tensor:
    """``linear`` with a 4-bit weight (``m3_linear4``): ``x @ W.T (+ residual)`` for the few rows
    of a decode step, ``W = (code - zero) * scale`` a ``Weight4``.

    ``x [M, K]`` (``M <= 256``) bfloat16 or float16; ``residual`` and ``out`` ``[M, N]`` of that
    dtype. Sums are FP32, the residual is added to them and the result rounded once. With
    ``norm_weight [K]`` (taken in ``x``'s dtype) ``x`` is first RMS-normalised, as
    ``F.rms_norm(x.float(), (K,), norm_weight.float(), norm_eps)``, its rows not rounded to 16
    bits. An infinity in a row of ``x`` makes its row of the result NaN. No backward.
    """
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, residual, norm_weight)
    index = x.get_device()
    if index < 0 or any([t is not None and t.get_device() != index
                         for t in (residual, out, norm_weight)]):
        _require_device(x, residual, out, norm_weight)
    if torch.is_grad_enabled():
        _require_inference(x, residual, norm_weight)
    if not linear4_supported(x, weight):
        raise ValueError(f"linear4: unsupported operands x {tuple(x.shape)} {x.dtype} on "
                         f"{x.device}, weight {weight.shape} on {weight.device}")
    m, (n, k), dtype = x.shape[0], weight.shape, x.dtype
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (t.shape != (m, n) or t.dtype != dtype):
            raise ValueError(f"linear4: {name} must be [{m}, {n}] {dtype}, got "
                             f"{tuple(t.shape)} {t.dtype}")
    if norm_weight is not None:
        if norm_weight.shape != (k,):
            raise ValueError(f"linear4: norm_weight must be [{k}]")
        if norm_weight.dtype != dtype:
            norm_weight = norm_weight.detach().to(dtype)
        norm_weight = _aligned16(norm_weight)
    x = _aligned16(x)
    residual, given = _inner(residual), out is not None
    if not given:
        out = x.new_empty((m, n))
    elif n > 1 and out.stride(1) != 1:
        raise ValueError("linear4: out needs a unit inner stride")
    code = _hip.dtype_code(dtype)
    none = _hip.NO_TENSOR
    _hip.launch("m3_linear4", _hip.LINEAR4.pack(
        m, n, k, code, _hip.dtype_code(weight.dtype), weight.group, norm_eps,
        weight.codes.data_ptr(), weight.scales.data_ptr(),
        0 if weight.zeros is None else weight.zeros.data_ptr(),
        x.data_ptr(), code, 0, *x.stride(), 0, 0, 0,
        *(none if norm_weight is None else (norm_weight.data_ptr(), code, 0, 1, 0, 0, 0, 0)),
        *(none if residual is None else (residual.data_ptr(), code, 0, *residual.stride(), 0, 0, 0)),
        out.data_ptr(), code, 0, *out.stride(), 0, 0, 0), index)
    if given:
        _written(out)
    return out


# --------------------------------------------------------------------------- 8-bit projections


def _device_index(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The one ROCm device that all of them are on; else a ``RuntimeError`` says which is not."""
    index = first.get_device()
    if index < 0 or any([t is not None and t.get_device() != index for t in others]):
        _require_device(first, *others)
    return index


class Rows8:
    """Rows ``[..., K]`` in 8 bits: ``codes`` int8, -128 to 127, with one FP32 scale each (``scales
    [...]``); a row is ``code * scale``. ``quantize8_rows`` and ``rms_norm8`` make them, ``linear8`` multiplies
    them. Codes from elsewhere are taken as they are where their columns lie side by side and their rows
    evenly apart, else copied.
    """

    # _ld: bytes between rows; _memory: the int8 tensor of both (codes, then scales), or of given codes
    # with _given, their scales
    __slots__ = ("shape", "_rows", "_ld", "_memory", "_given")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor) -> None:
        shape = codes.shape
        if len(shape) < 1 or codes.dtype != torch.int8 or shape[-1] == 0:
            raise ValueError("codes must be int8 of shape [..., K]")
        if scales.shape != shape[:-1] or scales.dtype != torch.float32:
            raise ValueError(f"scales must be float32 of shape {tuple(shape[:-1])}")
        if scales.device != codes.device:
            raise ValueError("codes and scales must be on the same device")
        width, rows = shape[-1], scales.numel()
        if width > _hip.LINEAR8_MAX_K:
            raise ValueError(f"rows of {width}: at most {_hip.LINEAR8_MAX_K}")
        scales, ld = scales.contiguous(), width
        if not codes.is_contiguous():
            codes = codes.reshape(-1, width)
            if codes.stride(1) != 1 and width > 1 or not width <= codes.stride(0) <= 1 << 22:
                codes = codes.contiguous()
            ld = codes.stride(0)
        self.shape, self._rows, self._ld, self._memory, self._given = shape, rows, ld, codes, scales

    @classmethod
    def _of(cls, memory: torch.Tensor, shape: torch.Size, rows: int, ld: int) -> Rows8:
        """Of ``memory``, what a kernel writes: ``[rows, ld]`` bytes of codes, then the scales."""
        self = object.__new__(cls)
        self.shape, self._rows, self._ld, self._memory, self._given = shape, rows, ld, memory, None
        return self

    def _block(self) -> tuple[int, int, int]:
        """Where the codes lie, the bytes between rows, where the scales lie."""
        at = self._memory.data_ptr()
        return (at, self._ld, at + self._rows * self._ld if self._given is None
                else self._given.data_ptr())

    @property
    def device(self) -> torch.device:
        return self._memory.device

    @property
    def codes(self) -> torch.Tensor:
        """The codes, int8 ``[..., K]``."""
        held, shape = self._memory, self.shape
        if self._given is None:
            held = held[:self._rows * self._ld].view(self._rows, self._ld)
        if held.shape == shape:
            return held
        held = held[:, :shape[-1]]
        return held[0] if len(shape) == 1 else held.unflatten(0, shape[:-1])

    @property
    def scales(self) -> torch.Tensor:
        """The scales, FP32 ``[...]``."""
        if self._given is not None:
            return self._given
        return self._memory[self._rows * self._ld:].view(torch.float32).view(self.shape[:-1])

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The rows ``[..., K]`` as ``code * scale``, one product in FP32 rounded to ``dtype``
        (``m3_rows8_values``; rows off the GPU in torch)."""
        given, memory, shape, rows = self._given, self._memory, self.shape, self._rows
        if forward_ad._current_level >= 0:
            _refuse_tangents(given)
        if given is not None and torch.is_grad_enabled():
            _require_inference(given)
        index = memory.get_device()
        if dtype not in _FLOAT_DTYPES or index < 0:
            return torch.mul(self.codes, self.scales.unsqueeze(-1)).to(dtype)
        out = memory.new_empty(shape, dtype=dtype)
        if rows:
            width = shape[-1]
            _hip.launch("m3_rows8_values", _hip.ROWS8_VALUES.pack(
                rows, width, *self._block(),
                out.data_ptr(), _hip.dtype_code(dtype), 0, width, 1, 0, 0, 0), index)
        return out


class Weight8:
    """An ``nn.Linear`` weight ``[N, K]`` held in 8 bits, laid out for ``linear8``: ``codes [N, K]`` int8 with
    one FP32 scale a row (an output channel); the weight is ``code * scale``. Both are copied into the kernel's
    tiles once, here (``m3_linear8``'s layout); later changes to them are not seen.
    """

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor) -> None:
        if codes.ndim != 2 or codes.dtype != torch.int8 or codes.numel() == 0:
            raise ValueError("codes must be int8 of shape [N, K]")
        n, k = codes.shape
        if scales.shape != (n,) or scales.dtype != torch.float32:
            raise ValueError(f"scales must be float32 of shape {(n,)}")
        if scales.device != codes.device:
            raise ValueError("codes and scales must be on the same device")
        if k > _hip.LINEAR8_MAX_K:
            raise ValueError(f"rows of {k}: at most {_hip.LINEAR8_MAX_K}")
        self.shape, self.device = (n, k), codes.device
        tn, tk = -(-n // 64), 2 * -(-k // 128)
        q = torch.nn.functional.pad(codes.detach(), (0, 64 * tk - k, 0, 64 * tn - n))
        # rows of a tile: [quarter's high bit, 4, quarter's low bit, 4]; columns: [lane group, byte]
        q = q.view(tn, 2, 4, 2, 4, tk, 4, 16).permute(0, 5, 1, 3, 6, 2, 4, 7)
        self.q = q.reshape(tn, tk, 4, 64, 16).contiguous()
        self.scales = torch.nn.functional.pad(scales.detach(), (0, 64 * tn - n))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The weight ``[N, K]`` as ``code * scale``, one product in FP32 rounded to ``dtype``."""
        n, k = self.shape
        tn, tk = self.q.shape[:2]
        q = self.q.view(tn, tk, 2, 2, 4, 4, 4, 16).permute(0, 2, 5, 3, 6, 1, 4, 7)
        q = q.reshape(64 * tn, 64 * tk)[:n, :k]
        return torch.mul(q, self.scales[:n].unsqueeze(1)).to(dtype)


def quantize8(weight: torch.Tensor) -> Weight8:
    """``weight [N, K]`` rounded to 8 bits, each row as ``quantize8_rows`` does one: its greatest
    magnitude has code 127 or -127, and codes are the exact quotients' nearest, ties to even."""
    if weight.ndim != 2 or weight.dtype not in _FLOAT_DTYPES or weight.numel() == 0:
        raise ValueError("weight must be a floating [N, K] tensor")
    weight = weight.detach()
    most = weight.abs().amax(1, keepdim=True).double()
    if not bool(torch.isfinite(most).all()):
        raise ValueError("quantize8: the weight holds NaN or infinities")
    # in 64 bits the product is exact and the quotient on the right side of half a code
    codes = (127 * weight.double() / torch.where(most > 0, most, 1.0)).round().to(torch.int8)
    return Weight8(codes, most.squeeze(1).float() / 127)


def _row_tensor(t: torch.Tensor | None, width: int) -> tuple[object, tuple[int, ...]]:
    """``[..., width]`` as rows: what has to stay alive across the call, and the values of its
    descriptor."""
    if t is None:
        return None, _hip.NO_TENSOR
    if t.is_contiguous():
        return t, (t.data_ptr(), _hip.dtype_code(t.dtype), 0, width, 1, 0, 0, 0)
    t = _inner(t.reshape(-1, width))
    return t, (t.data_ptr(), _hip.dtype_code(t.dtype), 0, *t.stride(), 0, 0, 0)


def _rows8(x, weight, eps, add, keep_sum, index) -> tuple[Rows8, torch.Tensor | None]:
    shape = x.shape
    width = shape[-1]
    rows, ld = x.numel() // width, -(-width // 64) * 64
    memory = x.new_empty(rows * (ld + 4), dtype=torch.int8)
    total = x.new_empty(shape) if keep_sum else None
    if rows:
        at = memory.data_ptr()
        held_x, block_x = _row_tensor(x, width)
        held_add, block_add = _row_tensor(add, width)
        _hip.launch("m3_rows8", _hip.ROWS8.pack(
            rows, width, eps, 0, *block_x, *block_add,
            *(_hip.NO_TENSOR if weight is None else
              (weight.data_ptr(), _hip.dtype_code(weight.dtype), 0, 1, 0, 0, 0, 0)),
            *_row_tensor(total, width)[1], at, ld, at + rows * ld), index)
        del held_x, held_add
    return Rows8._of(memory, shape, rows, ld), total


def _check_rows8(name: str, x: torch.Tensor) -> None:
    if x.ndim < 1 or x.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"{name}: x must be float32, bfloat16 or float16 of shape [..., K]")
    if not 0 < x.shape[-1] <= _hip.LINEAR8_MAX_K:
        raise ValueError(f"{name}: rows of {x.shape[-1]}: 1 to {_hip.LINEAR8_MAX_K}")


def quantize8_rows(x: torch.Tensor) -> Rows8:
    """Rows ``[..., K]`` rounded to 8 bits with a scale each (``m3_rows8``): ``scale = max|x| / 127``,
    ``code = rint(127 x / max|x|)`` of the exact quotient, ties to even.

    FP32, bfloat16 or float16, any strides. A row of zeros has codes and scale 0; one that holds an
    infinity or NaN has codes 0 and scale NaN. No backward.
    """
    _check_rows8("quantize8_rows", x)
    if forward_ad._current_level >= 0:
        _refuse_tangents(x)
    index = _device_index(x)
    if torch.is_grad_enabled():
        _require_inference(x)
    return _rows8(x, None, 0.0, None, False, index)[0]


def rms_norm8(x: torch.Tensor, weight: torch.Tensor, eps: float = NORM_EPS, *,
              add: torch.Tensor | None = None, keep_sum: bool = False):
    """``rms_norm`` with its output in 8 bits (``m3_rows8``): ``s = x + add`` (or ``x``), then
    ``quantize8_rows(F.rms_norm(s, (K,), weight.to(s.dtype), eps))`` with the norm's rows not rounded in
    between. Returns ``(Rows8, s)`` with ``s`` only when ``keep_sum`` (``add`` given).

    Rows of any K and strides: an FP32 ``x`` with an ``add`` of any dtype, or a 16-bit ``x`` with one of its
    own. The norm's factor is in the scale, not in the codes: ``code = rint(127 p / max|p|)`` with ``p = s *
    weight``. Rows of zeros, infinities and NaN as in ``quantize8_rows``; with ``eps = 0`` zeros alone give a
    scale of NaN, as ``F.rms_norm`` gives NaN. No backward.
    """
    _check_rows8("rms_norm8", x)
    if weight.shape != x.shape[-1:] or weight.dtype not in _FLOAT_DTYPES:
        raise ValueError(f"rms_norm8: weight must be floating of shape {tuple(x.shape[-1:])}")
    if add is not None and (add.shape != x.shape or add.dtype not in _FLOAT_DTYPES or (
            x.dtype != torch.float32 and add.dtype != x.dtype)):
        raise ValueError(f"rms_norm8: add must have x's shape {tuple(x.shape)}, and x's dtype unless "
                         "x is float32")
    if keep_sum and add is None:
        raise ValueError("rms_norm8: keep_sum needs add")
    if not eps >= 0:
        raise ValueError("rms_norm8: eps must be >= 0")
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, add)
    index = _device_index(x, weight, add)
    if torch.is_grad_enabled():
        _require_inference(x, weight, add)
    return _rows8(x, _inner(weight), eps, add, keep_sum, index)


def linear8(rows: Rows8, weight: Weight8, residual: torch.Tensor | None = None, *,
            out: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The product of rows and a weight in 8 bits, ``rows @ W.T (+ residual)`` (``m3_linear8``).

    ``rows [..., K]`` any number of them, one token's or a prompt's; the result ``[..., N]`` has ``dtype``
    FP32, bfloat16 or float16 (default: that of ``out`` or ``residual``, else bfloat16), which
    ``residual`` and ``out`` share. Sums are exact in 32-bit integers; scales and residual meet them in FP32, which
    is rounded once. ``out`` may be ``residual``. A row whose scale is NaN gives NaN. No backward.
    """
    if dtype is None:
        given = out if out is not None else residual
        dtype = torch.bfloat16 if given is None else given.dtype
    if dtype not in _FLOAT_DTYPES:
        raise ValueError("linear8: dtype must be float32, bfloat16 or float16")
    n, k = weight.shape
    if rows.shape[-1] != k:
        raise ValueError(f"linear8: rows {tuple(rows.shape)} do not fit weight {weight.shape}")
    shape = (*rows.shape[:-1], n)
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (t.shape != shape or t.dtype != dtype):
            raise ValueError(f"linear8: {name} must be {shape} {dtype}, got {tuple(t.shape)} {t.dtype}")
    if forward_ad._current_level >= 0:
        _refuse_tangents(residual, rows._given)
    index = _device_index(rows._memory, weight.q, residual, out)
    if torch.is_grad_enabled():
        _require_inference(residual, rows._given)
    given, m = out is not None, rows._rows
    if not given:
        out = rows._memory.new_empty(shape, dtype=dtype)
    flat = out if out.is_contiguous() else out.view(-1, n)
    if given and flat is not out and (m > 1 and flat.stride(0) < n or n > 1 and flat.stride(1) != 1):
        raise ValueError("linear8: out needs a unit inner stride and rows of its own")
    if m:
        ws = None
        codes, ld, scales = rows._block()
        exact = rows._given is not None
        residual, block = _row_tensor(residual, n)
        values = (m, n, k, _hip.dtype_code(dtype), exact, codes, ld, scales, weight.q.data_ptr(),
                  weight.scales.data_ptr(), *block, *_row_tensor(flat, n)[1])
        if exact and (codes % 16 or ld % 16 or k % 16):
            size = _hip.need("m3_linear8_workspace_size", _hip.LINEAR8.pack(*values, 0, 0))
            ws = rows._memory.new_empty(size) if size else None
        _hip.launch("m3_linear8", _hip.LINEAR8.pack(
            *values, *((0, 0) if ws is None else (ws.data_ptr(), ws.numel()))), index)
        del ws, residual
    if given:
        _written(out)
    return out


# --------------------------------------------------------------------------- gated recurrence


def _validate_gated(x, decay, gate, rate, state, state_name) -> None:
    if decay.shape != x.shape or (gate is not None and gate.shape != x.shape):
        raise ValueError("decay and gate must have the shape of x")
    if x.dtype not in _FLOAT_DTYPES or decay.dtype != x.dtype or (
            gate is not None and gate.dtype != x.dtype):
        raise ValueError("x, decay and gate must share one dtype: float32, bfloat16 or float16")
    if (gate is None) != (rate is None):
        raise ValueError("gate and rate must be provided together")
    width = x.shape[-1]
    if rate is not None and (rate.shape != (width,) or not rate.is_floating_point()):
        raise ValueError(f"rate must be a floating tensor of shape {(width,)}")
    if state is not None and (state.shape != (x.shape[0], width) or state.dtype != torch.float32):
        raise ValueError(f"{state_name} must be float32 of shape {(x.shape[0], width)}")


_NO_GATES = 2 * _hip.NO_TENSOR


def _tokens(t: torch.Tensor | None) -> torch.Tensor | None:
    """``[B, L, C]`` with a unit inner stride and tokens as near as the kernels' 32-bit offsets
    ask (copied only if it has not)."""
    t = _inner(t)
    if t is None or t.stride(1) <= 1 << 24:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _rate32(rate: torch.Tensor | None) -> torch.Tensor | None:
    if rate is None or (rate.dtype == torch.float32 and rate.is_contiguous()):
        return rate
    return rate.float().contiguous()


def _packed(t: torch.Tensor | None, code: int = 0):
    """A tensor of 1 to 3 axes as the values of its descriptor."""
    if t is None:
        return _hip.NO_TENSOR
    strides = t.stride()
    return (t.data_ptr(), code, 0, *strides, *(0,) * (5 - len(strides)))


def _gated_inputs(x, decay, gate, rate, state, lengths, reset):
    """The inputs of a gated scan [B, L, C] as the first values of its argument block."""
    code = _hip.dtype_code(x.dtype)
    return (*x.shape, code, *_packed(x, code), *_packed(decay, code), *_packed(gate, code),
            *_packed(rate), *_packed(state), 0 if lengths is None else lengths.data_ptr(),
            *((0, 0) if reset is None else (reset.data_ptr(), reset.stride(0))))


def _gated_forward(x, decay, gate, rate, state, lengths, reset, want_carry):
    batch, length, width = x.shape
    device = x.device
    out = x.new_empty(x.shape)
    if x.numel() == 0:
        return out, (torch.zeros(batch, width, dtype=torch.float32, device=device)
                     if state is None else state.clone()), None
    final = torch.empty((batch, width), dtype=torch.float32, device=device)
    carry = torch.empty((-(-length // _hip.GATED_TILE), batch, width), dtype=torch.float32,
                        device=device) if want_carry else None
    values = (*_gated_inputs(x, decay, gate, rate, state, lengths, reset),
              *_packed(out, _hip.dtype_code(x.dtype)), *_packed(final), *_packed(carry))
    block, ws = _hip.GATED_SCAN.pack(*values, 0, 0), None
    size = _hip.need("m3_gated_scan_workspace_size", block)
    if size:
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        block = _hip.GATED_SCAN.pack(*values, ws.data_ptr(), size)
    _hip.launch("m3_gated_scan", block, device.index)
    del ws
    return out, final, carry


class _GatedScan(torch.autograd.Function):
    """``gated_scan`` under autograd: the forward call also leaves the state after every
    ``GATED_TILE`` tokens, from which the backward call recomputes the states between."""

    @staticmethod
    def forward(ctx, x, decay, gate, rate, state, lengths, reset):
        out, final, carry = _gated_forward(x, decay, gate, rate, state, lengths, reset, True)
        ctx.save_for_backward(x, decay, gate, rate, state, lengths, reset, carry)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        x, decay, gate, rate, state, lengths, reset, carry = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 7
        if x.numel() == 0:
            if state is not None and dfinal is None:
                dfinal = torch.zeros_like(state)
            return (*(None if t is None else torch.zeros_like(t) for t in (x, decay, gate, rate)),
                    None if state is None else dfinal, None, None)
        code, none = _hip.dtype_code(x.dtype), _hip.NO_TENSOR
        dout = x.new_zeros(x.shape) if dout is None else _tokens(dout)
        dfinal = _inner(dfinal)
        dx, ddecay = x.new_empty(x.shape), x.new_empty(x.shape)
        dgate = drate = dstate = None
        if gate is not None:
            dgate, drate = x.new_empty(x.shape), torch.empty_like(rate)
        if state is not None:
            dstate = torch.empty_like(state, memory_format=torch.contiguous_format)
        inputs = (*_gated_inputs(x, decay, gate, rate, state, lengths, reset), *none, *none,
                  *_packed(carry))
        grads = (*_packed(dout, code), *_packed(dfinal), *_packed(dx, code),
                 *_packed(ddecay, code), *_packed(dgate, code), *_packed(drate),
                 *_packed(dstate))
        size = _hip.need("m3_gated_scan_bwd_workspace_size",
                         _hip.GATED_SCAN_BWD.pack(*inputs, 0, 0, *grads))
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        _hip.launch("m3_gated_scan_bwd",
                    _hip.GATED_SCAN_BWD.pack(*inputs, ws.data_ptr(), size, *grads), x.get_device())
        return dx, ddecay, dgate, drate, dstate, None, None


def gated_scan(x: torch.Tensor, decay: torch.Tensor, gate: torch.Tensor | None = None,
               rate: torch.Tensor | None = None, *, initial_state: torch.Tensor | None = None,
               lengths: torch.Tensor | None = None, reset: torch.Tensor | None = None):
    """A gated linear recurrence over ``[B, L, C]``, one FP32 state per channel (``m3_gated_scan``).

    Without ``gate`` and ``rate``, ``decay`` holds log decays, at most 0 (factors are multiplied over
    tiles of tokens, so positive ones can give NaN where the recurrence is finite): ``h_t =
    exp(decay_t) h_{t-1} + x_t``. With them ``decay`` and ``gate`` hold logits and ``rate [C]`` (>=
    0) the log decay of an open gate: ``a_t = exp(-rate sigmoid(decay_t))``, ``h_t = a_t h_{t-1} +
    sqrt(1 - a_t^2) sigmoid(gate_t) x_t``. ``x``, ``decay`` and ``gate`` share one dtype and may be
    slices of one projection. Returns ``(out [B, L, C] = h in x's dtype, final_state [B, C] FP32)``.

    ``initial_state [B, C]`` FP32 continues a sequence. ``lengths [B]`` (integers; clamped to 0..L)
    ends each row of a padded batch: past its end ``out`` is 0 and the state stays, whatever the
    padding holds. ``reset [B, L]`` (bool) marks tokens that start from an empty state, as the
    first token of each document in a packed row does. The gate form is the RG-LRU recurrence, except
    that the published one drops the factor ``sqrt(1 - a_t^2)`` at tokens that begin a sequence (the
    first and reset ones); here they have it too.

    Unlike the Mamba-3 calls of this module this one has a backward pass: gradients reach ``x``,
    ``decay``, ``gate``, ``rate`` and ``initial_state`` (once: no second derivatives, none in
    forward mode).
    """
    if x.ndim != 3:
        raise ValueError("x must have shape [B, L, C]")
    _validate_gated(x, decay, gate, rate, initial_state, "initial_state")
    batch, length, width = x.shape
    if lengths is not None and (lengths.shape != (batch,) or
                                lengths.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"lengths must be int32 or int64 of shape {(batch,)}")
    if reset is not None and (reset.shape != (batch, length) or
                              reset.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"reset must be bool of shape {(batch, length)}")
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, decay, gate, rate, initial_state)
    index = x.get_device()
    if index < 0 or any([t is not None and t.get_device() != index for t in
                         (decay, gate, rate, initial_state, lengths, reset)]):
        _require_device(x, decay, gate, rate, initial_state, lengths, reset)
    rate = _rate32(rate)
    if lengths is not None and (lengths.dtype != torch.int32 or not lengths.is_contiguous()):
        lengths = lengths.clamp(0, length).to(torch.int32).contiguous()
    x, decay, gate = _tokens(x), _tokens(decay), _tokens(gate)
    state, reset = _inner(initial_state), _inner(reset)
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad
                                        for t in (x, decay, gate, rate, state)]):
        return _GatedScan.apply(x, decay, gate, rate, state, lengths, reset)
    return _gated_forward(x, decay, gate, rate, state, lengths, reset, False)[:2]


def gated_step(x: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
               gate: torch.Tensor | None = None, rate: torch.Tensor | None = None, *,
               inplace: bool = False):
    """One token of ``gated_scan``: ``x``, ``decay``, ``gate`` ``[B, C]``, ``state [B, C]`` FP32.

    Returns ``(out [B, C], state')``. ``inplace`` writes the new state into ``state`` (the static
    cache of a captured decode step), which then needs a unit inner stride. No backward.
    """
    if x.ndim != 2:
        raise ValueError("x must have shape [B, C]")
    _validate_gated(x, decay, gate, rate, state, "state")
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, decay, gate, rate, state)
    index = x.get_device()
    if index < 0 or decay.get_device() != index or state.get_device() != index or (
            gate is not None and not gate.get_device() == rate.get_device() == index):
        _require_device(x, decay, gate, rate, state)
    if torch.is_grad_enabled():
        _require_inference(x, decay, gate, rate, state)
    batch, width = x.shape
    if inplace and ((width > 1 and state.stride(1) != 1) or
                    (batch > 1 and state.stride(0) < width)):
        raise ValueError("state must have a unit innermost stride and rows of its own to be "
                         "updated in place")
    out = x.new_empty((batch, width))
    new = state if inplace else state.new_empty((batch, width))
    if batch == 0 or width == 0:
        return out, new
    x, decay, state = _inner(x), _inner(decay), _inner(state)
    code, none, gates = _hip.dtype_code(x.dtype), _hip.NO_TENSOR, _NO_GATES
    if gate is not None:
        gate, rate = _inner(gate), _rate32(rate)
        gates = (gate.data_ptr(), code, 0, gate.stride(0), 0, 1, 0, 0,
                 rate.data_ptr(), 0, 0, 1, 0, 0, 0, 0)
    _hip.launch("m3_gated_scan", _hip.GATED_SCAN.pack(
        batch, 1, width, code,
        x.data_ptr(), code, 0, x.stride(0), 0, 1, 0, 0,
        decay.data_ptr(), code, 0, decay.stride(0), 0, 1, 0, 0,
        *gates,
        state.data_ptr(), 0, 0, state.stride(0), 1, 0, 0, 0,
        0, 0, 0,
        out.data_ptr(), code, 0, width, 0, 1, 0, 0,
        new.data_ptr(), 0, 0, new.stride(0), 1, 0, 0, 0,
        *none, 0, 0), index)
    if inplace:
        _written(new)
    return out, new


__all__ = ["heavy_tail_activation", "mamba3_scan", "mamba3_step", "fused_step", "chunk_state",
           "ScanCall", "scan_projection", "step_projection", "split_projection", "linear",
           "linear_supported", "rms_norm", "rms_norm_supported", "gated_scan", "gated_step",
           "Weight4", "quantize4", "linear4", "linear4_supported", "Rows8", "Weight8", "quantize8",
           "quantize8_rows", "rms_norm8", "linear8"]
