"""The gated linear recurrence in 64 bits, token by token, and how far FP32 arithmetic may be from it.

``scan`` is the definition, in double and differentiable by torch. ``bounds`` follows the same recurrences for the
rounding errors of an FP32 evaluation: with u = 2^-24 (half a step of FP32) every product, sum,
reciprocal, root and exponential is taken as off by at most 2 u of its value (the hardware exp2,
rcp and rsq are good to 1 ulp = 2 u), and arguments' errors are carried through.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24


def _masks(x, lengths, reset):
    batch, length = x.shape[:2]
    valid = torch.ones(batch, length, 1, dtype=torch.bool)
    if lengths is not None:
        valid = (torch.arange(length) < lengths.cpu().long().clamp(0, length)[:, None])[..., None]
    fresh = torch.zeros(batch, length, 1, dtype=torch.bool)
    if reset is not None:
        fresh = (reset.cpu() != 0)[..., None]
    return valid, fresh & valid


def coefficients(decay, gate, rate):
    """log a, s = sqrt(1 - a^2) (1 in the given form) and the two sigmoids, in double."""
    decay = decay.double()
    if gate is None:
        return decay, torch.ones_like(decay), None, torch.ones_like(decay)
    p, q = torch.sigmoid(decay), torch.sigmoid(gate.double())
    log_a = -rate.double() * p
    return log_a, torch.sqrt(-torch.expm1(2 * log_a)), p, q


def scan(x, decay, gate=None, rate=None, state=None, lengths=None, reset=None):
    """(y, final) in double; inputs on the CPU. Masked inputs never enter a product."""
    valid, fresh = _masks(x, lengths, reset)
    zero = torch.zeros((), dtype=torch.float64)
    x = torch.where(valid, x.double(), zero)
    decay = torch.where(valid, decay.double(), zero)
    gate = None if gate is None else torch.where(valid, gate.double(), zero)
    log_a, s, _, q = coefficients(decay, gate, rate)
    a, b = torch.where(valid, torch.exp(log_a), 1.0), torch.where(valid, s * q * x, zero)
    h = torch.zeros(x.shape[0], x.shape[2], dtype=torch.float64) if state is None else state.double()
    ys = []
    for t in range(x.shape[1]):
        h = torch.where(fresh[:, t], zero, h)
        h = a[:, t] * h + b[:, t]
        ys.append(torch.where(valid[:, t], h, zero))
    return torch.stack(ys, 1), h


def bounds(x, decay, gate=None, rate=None, state=None, lengths=None, reset=None, dy=None,
           dfinal=None):
    """Absolute error bounds of an FP32 evaluation, by output name (finite valid inputs)."""
    valid, fresh = _masks(x, lengths, reset)
    zero = torch.zeros((), dtype=torch.float64)
    x, decay = (torch.where(valid, t.double(), zero) for t in (x, decay))
    gate = None if gate is None else torch.where(valid, gate.double(), zero)
    log_a, s, p, q = coefficients(decay, gate, rate)
    a = torch.where(valid, torch.exp(log_a), 1.0)
    if gate is None:
        ea = U * (2 + 3 * log_a.abs())  # exp2's own step, its argument's product
        ew = torch.zeros_like(ea)
        ep = eq = einv = ew
    else:
        # sigmoid: exp2's argument 1.45 |r| u, exp2, the sum, rcp and a product: 2 u each
        ep, eq = U * (8 + 1.5 * decay.abs()), U * (8 + 1.5 * gate.abs())
        elog = ep + 4 * U                       # of log a, relative
        ea = 2 * U + log_a.abs() * elog
        # 1 - a^2: near 0 a series of relative error elog + 8 u (its 4 steps and truncation);
        # else a difference of at least 0.117, its terms off by 2 ea + 4 u
        v = s * s
        ev = torch.where(2 * log_a > -0.126, elog + 8 * U, (2 * ea + 4 * U) * a * a / v + 2 * U)
        ev = torch.where(v > 0, ev, zero)
        es = 0.5 * ev + 4 * U
        einv = es
        ew = es + eq + 2 * U
    w = s * q
    b = torch.where(valid, w * x, zero)
    ea, ew = torch.where(valid, ea, zero), torch.where(valid, ew, zero)
    # h: |h| <= m; each token adds the error of its factor, its input and two roundings. Products
    # of factors formed ahead of the state (a tile's) round once more a token and a fold: 4 u m
    # in place of 2 u.
    batch, length, width = x.shape
    m = torch.zeros(batch, width, dtype=torch.float64) if state is None else state.double().abs()
    e = torch.zeros_like(m)
    before_m, before_e, ys = [], [], []
    for t in range(length):
        m, e = (torch.where(fresh[:, t], zero, v) for v in (m, e))
        before_m.append(m)
        before_e.append(e)
        e = a[:, t] * (e + ea[:, t] * m)
        m = a[:, t] * m + b[:, t].abs()
        e = e + (ew[:, t] + 2 * U) * b[:, t].abs() + 4 * U * m
        ys.append(torch.where(valid[:, t], e, zero))
    out = dict(y=torch.stack(ys, 1), final=e)
    if dy is None:
        return out
    dy = torch.where(valid, dy.double(), zero)
    m = torch.zeros(batch, width, dtype=torch.float64) if dfinal is None else dfinal.double().abs()
    e = torch.zeros_like(m)
    names = ("dx", "ddecay", "dgate")
    grads = {n: torch.zeros_like(x) for n in names}
    rate_e = torch.zeros(width, dtype=torch.float64)
    rate_v = torch.zeros(width, dtype=torch.float64)
    for t in range(length - 1, -1, -1):
        live = valid[:, t]
        dm = m + dy[:, t].abs()
        de = e + 2 * U * dm
        hm, he = before_m[t], before_e[t]
        at, wt, st, qt, xt = a[:, t], w[:, t], s[:, t], q[:, t], x[:, t].abs()
        grads["dx"][:, t] = torch.where(live, wt * (de + dm * (ew[:, t] + 2 * U)), zero)
        carry_v, carry_e = at * hm, at * (he + hm * (ea[:, t] + 2 * U))
        if gate is None:
            grads["ddecay"][:, t] = torch.where(live, de * carry_v + dm * (carry_e + 2 * U * carry_v),
                                                zero)
        else:
            inv = torch.where(st > 0, 1 / st, zero)
            slope = qt * xt * at * at * inv
            slope_e = slope * (eq[:, t] + 2 * ea[:, t] + einv[:, t] + 8 * U)
            value, err = carry_v + slope, carry_e + slope_e
            log_v = dm * value
            log_e = de * value + dm * (err + 4 * U * value)
            pp, qq = p[:, t] * (1 - p[:, t]), qt * (1 - qt)
            grads["ddecay"][:, t] = torch.where(
                live, rate.double() * pp * (log_e + log_v * (2 * ep[:, t] + 8 * U)), zero)
            grads["dgate"][:, t] = torch.where(
                live, st * xt * qq * (de + dm * (es[:, t] + 2 * eq[:, t] + 8 * U)), zero)
            rate_e += torch.where(live, p[:, t] * (log_e + log_v * (ep[:, t] + 2 * U)), zero).sum(0)
            rate_v += torch.where(live, p[:, t] * log_v, zero).sum(0)
        e = at * (de + dm * (ea[:, t] + 4 * U))
        m = at * dm
        m, e = (torch.where(fresh[:, t], zero, v) for v in (m, e))
    # a token's sums run over at most a tile and its waves in FP32 (128 terms), then in 64 bits
    return out | grads | dict(drate=rate_e + 130 * 2 * U * rate_v, dstate=e)
