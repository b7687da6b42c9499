"""Operators over sequences with a state: the causal depthwise convolution
over a few tokens and the selective state space scan.

Elements are [sequences, tokens, channels], channels contiguous, tokens and
sequences any distance apart (slices of a projection's output are read in
place).  Activations are fp32 or bf16, all of one type; parameters, scan
states and their gradients fp32.  `lengths` (int32 [sequences]) marks a
padded batch: a position past its sequence's length is not read, changes no
state, and outputs and gradients are 0 there.  A sequence may be empty.

The state before the first token is a constant of the backward passes, as in
the recurrent layers (ops/rnn.py); the state after the last token has no
gradient.

As the other operators of this package (ops/core.py, ops/nn.py), these are no
autograd nodes: on the GPU an output does not require grad whatever the inputs
do.  Gradients come from the *_bwd functions; the node that calls them is
StateSpaceLayer's (ops/functional.py).

A scan's decays are good to 2^-21 of their exponent (approximate exponentials
of a rounded product): fp32 outputs and gradients are within 1e-6 of their
norm, some twice as far from the exact ones as with torch.exp.  A rate
exp(a_log) past fp32's largest value counts as that value.

GPU tensors run csrc/kernels/short_conv.cu and state_scan.cu, CPU tensors the
same formulas in torch.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .core import N, native


# ---------------------------------------------------------------- checks of the CPU path
def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _check(name, t, dtype, shape):
    _need(t.dtype == dtype, f"{name} is {t.dtype}, expected {dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")


def _check_rows(x, name):
    _need(x.dim() == 3, f"{name} is [sequences, tokens, channels], got {tuple(x.shape)}")
    _need(x.dtype in (torch.float32, torch.bfloat16), f"{name} is fp32 or bf16, got {x.dtype}")


def _counted(lengths, B, T):
    """[B, T, 1]: the positions that count (None: all)."""
    if lengths is None:
        return None
    _check("lengths", lengths, torch.int32, (B,))
    return (torch.arange(T)[None, :] < lengths.long()[:, None])[..., None]


def _where(counted, x):
    return x if counted is None else torch.where(counted, x, torch.zeros_like(x))


def _put(value, out, accumulate=False):
    if out is None:
        return value
    return out.add_(value) if accumulate else out.copy_(value)


# ---------------------------------------------------------------- short convolution
def _conv_check(x, weight, bias, state):
    _check_rows(x, "x")
    B, T, D = x.shape
    _need(weight.dim() == 2 and 2 <= weight.shape[1] <= 4, f"weight is [channels, 2 to 4 taps], got {tuple(weight.shape)}")
    k = weight.shape[1]
    _check("weight", weight, torch.float32, (D, k))
    if bias is not None:
        _check("bias", bias, torch.float32, (D,))
    if state is not None:
        _check("state", state, x.dtype, (B, k - 1, D))


def _conv_parts(x, weight, bias, state, lengths):
    """(which positions count, the tokens with the ones before them, the sums before the activation)."""
    _conv_check(x, weight, bias, state)
    (B, T, D), k = x.shape, weight.shape[1]
    counted = _counted(lengths, B, T)
    before = state.float() if state is not None else torch.zeros(B, k - 1, D)
    whole = torch.cat([before, _where(counted, x.float())], 1)
    pre = sum(weight[:, j] * whole[:, j:j + T] for j in range(k))
    return counted, whole, pre if bias is None else pre + bias


def short_conv_fwd(x, weight, bias=None, state=None, lengths=None, silu: bool = True, want_state: bool = False,
                   out_state=None):
    """y[t] = act(bias + sum_j weight[:, j] x[t - taps + 1 + j]) for weight
    [channels, taps] of 2 to 4 taps, act SiLU or none; x before the first token
    is `state` [sequences, taps - 1, channels], or zeros.  Returns (y, the
    state after the last token that counts, or None); `out_state` (which may be
    `state`) is filled with it."""
    if native(x):
        y, last = N().short_conv_fwd(x, weight, bias, state, lengths, silu, want_state, out_state)
        return y, last
    counted, whole, pre = _conv_parts(x, weight, bias, state, lengths)
    y = _where(counted, pre * torch.sigmoid(pre) if silu else pre).to(x.dtype)
    if not want_state and out_state is None:
        return y, None
    (B, T, D), k = x.shape, weight.shape[1]
    end = lengths.long().clamp(0, T) if lengths is not None else torch.full((B,), T)
    at = (end[:, None] + torch.arange(k - 1))[..., None].expand(-1, -1, D)
    last = torch.gather(whole, 1, at).to(x.dtype)
    if out_state is not None:
        _check("out_state", out_state, x.dtype, (B, k - 1, D))
    return y, _put(last, out_state)


def short_conv_bwd(x, weight, bias, dy, state=None, lengths=None, silu: bool = True, dx=None, dweight=None, dbias=None,
                   accumulate: bool = False):
    """Gradients (dx, dweight, dbias or None) of short_conv_fwd.  Those given
    are written whole; with `accumulate` the parameters' are added to."""
    if native(x):
        return tuple(N().short_conv_bwd(x, weight, bias, dy, state, lengths, silu, dx, dweight, dbias, accumulate))
    counted, whole, pre = _conv_parts(x, weight, bias, state, lengths)
    (B, T, D), k = x.shape, weight.shape[1]
    _check("dy", dy, x.dtype, (B, T, D))
    _need(not accumulate or (dweight is not None and (dbias is not None or bias is None)),
          "accumulate needs dweight (and dbias where there is a bias)")
    _need(bias is not None or dbias is None, "dbias without a bias")
    g = _where(counted, dy.float())
    if silu:
        p = torch.sigmoid(pre)
        g = _where(counted, g * p * (1 + pre * (1 - p)))
    after = torch.cat([g, torch.zeros(B, k - 1, D)], 1)
    gx = sum(weight[:, j] * after[:, k - 1 - j:k - 1 - j + T] for j in range(k)).to(x.dtype)
    gw = torch.stack([(g * whole[:, j:j + T]).sum((0, 1)) for j in range(k)], 1)
    gb = _put(g.sum((0, 1)), dbias, accumulate) if bias is not None else None
    return _put(gx, dx), _put(gw, dweight, accumulate), gb


def short_conv_step(x, weight, bias, state, silu: bool = True, out_state=None):
    """y of one token x [sequences, channels] of each sequence; `state`
    moves on by it in place, or into `out_state` where that is given."""
    if native(x):
        return N().short_conv_step(x, weight, bias, state, silu, out_state)
    y, _ = short_conv_fwd(x.unsqueeze(1), weight, bias, state=state, silu=silu,
                          out_state=state if out_state is None else out_state)
    return y.squeeze(1)


# ---------------------------------------------------------------- state space scan
class StateScanGrads(NamedTuple):
    du: torch.Tensor
    ddt: torch.Tensor
    da_log: torch.Tensor
    db: torch.Tensor
    dc: torch.Tensor
    dskip: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddt_bias: Optional[torch.Tensor]


SPAN = 16  # tokens between two kept states (kernels.h STATE_SCAN_SPAN)


def _scan_parts(u, dt, a_log, b, c, skip, z, dt_bias, lengths):
    _check_rows(u, "u")
    B, T, D = u.shape
    _need(a_log.dim() == 2 and 1 <= a_log.shape[1] <= 64, f"a_log is [channels, 1 to 64 states], got {tuple(a_log.shape)}")
    n = a_log.shape[1]
    _check("a_log", a_log, torch.float32, (D, n))
    _check("dt", dt, u.dtype, (B, T, D))
    _need(b.dim() in (3, 4), f"b is [sequences, tokens, (groups,) states], got {tuple(b.shape)}")
    groups = b.shape[2] if b.dim() == 4 else 1
    _need(groups >= 1 and D % groups == 0, f"{D} channels in {groups} groups")
    shape = (B, T, groups, n) if b.dim() == 4 else (B, T, n)
    _check("b", b, u.dtype, shape)
    _check("c", c, u.dtype, shape)
    for name, p in (("skip", skip), ("dt_bias", dt_bias)):
        if p is not None:
            _check(name, p, torch.float32, (D,))
    if z is not None:
        _check("z", z, u.dtype, (B, T, D))
    counted = _counted(lengths, B, T)
    raw = dt.contiguous().float() + (dt_bias if dt_bias is not None else 0.0)
    step = _where(counted, torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs())))
    wide = lambda v: _where(counted, v.contiguous().reshape(B, T, groups * n).float()).reshape(B, T, groups, 1, n)  # noqa: E731
    uf = _where(counted, u.contiguous().float())
    # (no further than fp32's lowest value: an infinity times a step of 0 is not a number)
    return counted, groups, raw, step, uf, wide(b), wide(c), -torch.exp(a_log).clamp(max=torch.finfo(torch.float32).max)


def _scan_states(step, u, a, b, groups, state, T):
    """h before every token and after the last, [B, G, D / G, N] each."""
    B, D = u.shape[0], u.shape[2]
    split = lambda v: v.reshape(B, groups, D // groups, 1)  # noqa: E731
    rate = a.reshape(groups, D // groups, a.shape[1])
    h = state.reshape(B, *rate.shape) if state is not None else torch.zeros(B, *rate.shape)
    hs = [h]
    for t in range(T):
        h = torch.exp(split(step[:, t]) * rate) * h + split(step[:, t] * u[:, t]) * b[:, t]
        hs.append(h)
    return hs


def state_scan_fwd(u, dt, a_log, b, c, skip=None, z=None, dt_bias=None, state=None, lengths=None,
                   want_state: bool = False, save: bool = False, out_state=None):
    """The selective state space scan

        s = softplus(dt + dt_bias)      h[t] = exp(-s exp(a_log)) h[t-1] + s u b[t]
        y = (sum over states of c h + skip u) silu(z)

    u, dt, z [sequences, tokens, channels]; b, c [sequences, tokens, states] or
    [..., groups, states], a group for each run of channels / groups channels;
    a_log [channels, states] (1 to 64 states); skip, dt_bias [channels]; state
    [sequences, channels, states], or zeros.  Without z there is no gate.
    Returns (y, the state after the last token that counts or None, with `save`
    what state_scan_bwd needs or None); `out_state` (which may be `state`) is
    filled with that state."""
    if native(u):
        return tuple(N().state_scan_fwd(u, dt, a_log, b, c, skip, z, dt_bias, state, lengths, want_state, save,
                                        out_state))
    counted, groups, _, step, uf, bf, cf, a = _scan_parts(u, dt, a_log, b, c, skip, z, dt_bias, lengths)
    B, T, D = u.shape
    if state is not None:
        _check("state", state, torch.float32, (B, D, a.shape[1]))
    if out_state is not None:
        _check("out_state", out_state, torch.float32, (B, D, a.shape[1]))
    hs = _scan_states(step, uf, a, bf, groups, state, T)
    y = torch.stack([(hs[t + 1] * cf[:, t]).sum(-1).reshape(B, D) for t in range(T)], 1) if T else torch.zeros(B, 0, D)
    if skip is not None:
        y = y + skip * uf
    if z is not None:
        zf = _where(counted, z.contiguous().float())
        y = y * zf * torch.sigmoid(zf)
    y = _where(counted, y).to(u.dtype)
    last = saved = None
    if save:
        kept = [h.reshape(B, D, a.shape[1]) for h in hs[:T:SPAN]]
        saved = torch.stack(kept, 1) if kept else torch.zeros(B, 0, D, a.shape[1])
    if want_state or out_state is not None:
        last = _put(hs[-1].reshape(B, D, a.shape[1]).clone(), out_state)
    return y, last, saved


def state_scan_bwd(u, dt, a_log, b, c, dy, saved, skip=None, z=None, dt_bias=None, lengths=None, du=None, ddt=None,
                   db=None, dc=None, dz=None, da_log=None, dskip=None, ddt_bias=None,
                   accumulate: bool = False) -> StateScanGrads:
    """Gradients of state_scan_fwd from its `saved`; None for operands that are
    not there.  Those given are written whole; with `accumulate` the parameters'
    (da_log, dskip, ddt_bias) are added to."""
    if native(u):
        return StateScanGrads(*N().state_scan_bwd(u, dt, a_log, b, c, skip, z, dt_bias, dy, saved, lengths, du, ddt, db,
                                                  dc, dz, da_log, dskip, ddt_bias, accumulate))
    counted, groups, raw, step, uf, bf, cf, a = _scan_parts(u, dt, a_log, b, c, skip, z, dt_bias, lengths)
    B, T, D = u.shape
    n = a.shape[1]
    _check("dy", dy, u.dtype, (B, T, D))
    _check("saved", saved, torch.float32, (B, (T + SPAN - 1) // SPAN, D, n))
    _need((z is not None or dz is None) and (skip is not None or dskip is None) and
          (dt_bias is not None or ddt_bias is None), "a gradient of an operand that is not there")
    _need(not accumulate or (da_log is not None and (dskip is not None or skip is None) and
                             (ddt_bias is not None or dt_bias is None)),
          "accumulate needs the parameters' gradients")
    hs = _scan_states(step, uf, a, bf, groups, saved[:, 0] if T else None, T)
    q = g_out = _where(counted, dy.contiguous().float())
    if z is not None:
        zf = _where(counted, z.contiguous().float())
        pz = torch.sigmoid(zf)
        q = g_out * zf * pz
    split = lambda v: v.reshape(B, groups, D // groups, 1)  # noqa: E731
    rate = a.reshape(groups, D // groups, n)
    carry = torch.zeros(B, groups, D // groups, n)
    into, through_a = torch.zeros(B, T, D), torch.zeros(B, T, D)
    gb, gc = torch.zeros(B, T, groups, n), torch.zeros(B, T, groups, n)
    ga = torch.zeros(groups, D // groups, n)
    pre = torch.zeros(B, T, D)
    for t in range(T - 1, -1, -1):
        g = cf[:, t] * split(q[:, t]) + carry
        gb[:, t] = (g * split(step[:, t] * uf[:, t])).sum(2)
        gc[:, t] = (hs[t + 1] * split(q[:, t])).sum(2)
        pre[:, t] = (hs[t + 1] * cf[:, t]).sum(-1).reshape(B, D)
        into[:, t] = (g * bf[:, t]).sum(-1).reshape(B, D)
        carry = g * torch.exp(split(step[:, t]) * rate)
        through = carry * hs[t]
        through_a[:, t] = (through * rate).sum(-1).reshape(B, D)
        ga += (through * split(step[:, t])).sum(0)
    slope = torch.sigmoid(raw)  # 0 for a step of 0, however large the rates are
    draw = _where(counted, torch.where(slope == 0, slope, (through_a + into * uf) * slope))
    gu = into * step + (q * skip if skip is not None else 0.0)
    gz = None
    if z is not None:
        full = pre + skip * uf if skip is not None else pre
        gz = _put((g_out * full * pz * (1 + zf * (1 - pz))).to(u.dtype), dz)
    shape = b.shape
    return StateScanGrads(
        _put(gu.to(u.dtype), du), _put(draw.to(u.dtype), ddt), _put((ga * rate).reshape(D, n), da_log, accumulate),
        _put(gb.to(u.dtype).reshape(shape), db), _put(gc.to(u.dtype).reshape(shape), dc),
        _put((q * uf).sum((0, 1)), dskip, accumulate) if skip is not None else None, gz,
        _put(draw.sum((0, 1)), ddt_bias, accumulate) if dt_bias is not None else None)


def state_scan_step(u, dt, a_log, b, c, state, skip=None, z=None, dt_bias=None, out_state=None):
    """One token of each sequence: u, dt, z [sequences, channels], b, c
    [sequences, states] or [sequences, groups, states].  Returns y; `state`
    moves on in place, or into `out_state` where that is given."""
    if native(u):
        return N().state_scan_step(u, dt, a_log, b, c, state, skip, z, dt_bias, out_state)
    y, _, _ = state_scan_fwd(u.unsqueeze(1), dt.unsqueeze(1), a_log, b.unsqueeze(1), c.unsqueeze(1), skip,
                             z.unsqueeze(1) if z is not None else None, dt_bias, state,
                             out_state=state if out_state is None else out_state)
    return y.squeeze(1)
