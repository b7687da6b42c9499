"""The short causal convolution and the selective state space scan in the cases
at their borders; the formulas in 64 bits and the tolerances are test_sequence_ops'."""
import math

import pytest
import torch

from dlvk_b200.ops import ssm
from test_sequence_ops import DEVICES, DTYPES, HALF, limits, near, run_scan, run_scan_bwd, scan_check, scan_inputs, scan_ref


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,G", [(1, 16, 1), (5, 16, 1), (23, 5, 1), (300, 16, 1), (40, 33, 2)])
def test_scan_of_rates_past_fp32(device, dtype, T, N, G):
    """exp(a_log) past fp32's largest value: a token of any length leaves nothing
    of the state, one of no length (masked, or behind its sequence) all of it.
    Decays of 0 have no error, so the tolerance is that of the other states."""
    p, dy, state, _ = scan_inputs(3, T, 24, N, G, dtype, device, T + N)
    p["dt"], p["dt_bias"] = p["dt"].clamp(-4, 4), p["dt_bias"].clamp(-4, 4)  # steps of 3e-4 and more
    p["a_log"] = p["a_log"].clamp(max=2.0)
    xmax = scan_ref(p, None, state, None)[3]
    p["a_log"][3:9] = 90.0
    p["a_log"][10, 0] = 500.0
    p["a_log"][11, 0] = math.inf
    short, long = limits(p, xmax)
    ref = dict(p, a_log=p["a_log"].clamp(max=600.0))  # (whose rates are finite in 64 bits)
    for n in (None, torch.tensor([T, T // 2, 0], dtype=torch.int32, device=device)):
        (y, h, g, _), (my, mh, mg, _) = (scan_ref(ref, dy, state, n, absolute=a) for a in (False, True))
        gy, gh, saved = run_scan(p, state=state, lengths=n, want_state=True, save=True)
        near(gy, y, my, short, "y")
        near(gh, h, mh, short, "state")
        grads = run_scan_bwd(p, dy, saved, lengths=n)
        for k in ("u", "dt", "a_log", "b", "c", "skip", "z", "dt_bias"):
            near(getattr(grads, "d" + k), g[k], mg[k], long, k)
    masked = dict(p, dt=torch.full_like(p["dt"], -math.inf))
    y, h, saved = run_scan(masked, state=state, want_state=True, save=True)
    assert torch.equal(h, state) and bool(torch.isfinite(y).all())
    assert all(bool(torch.isfinite(v).all()) for v in run_scan_bwd(masked, dy, saved))
    nan = dict(p, a_log=p["a_log"].clone())
    nan["a_log"][5] = math.nan
    y = run_scan(nan, state=state)[0]
    assert bool(torch.isnan(y[..., 5]).all()) and bool(torch.isfinite(y[..., 6:]).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [1, 3])
def test_scan_of_no_channels(device, dtype, G):
    """No channel reads b and c: their gradients are zeros, whatever was there."""
    p, dy, state, _ = scan_inputs(2, 19, 0, 5, G, dtype, device)
    y, last, saved = run_scan(p, state=state, want_state=True, save=True)
    assert y.shape == (2, 19, 0) and last.shape == (2, 0, 5)
    given = {k: torch.full_like(p["b"], 7.0) for k in ("db", "dc")}
    grads = run_scan_bwd(p, dy, saved, **given)
    assert not given["db"].any() and not given["dc"].any() and grads.da_log.shape == (0, 5)


def scan_ref_wide(p, dy, n, absolute=False):
    """The gradients of test_sequence_ops.scan_ref, from a state of zeros, for many
    sequences and tokens at once: in 64 bits where the tensors are.  With `absolute`
    the magnitudes of all products, and how far rounded decays and running sums
    move them: a decay of argument x is off by 2^-22 + 2^-21 x of itself, as in
    test_sequence_ops, a running sum by 2^-23 a token (its product and its sum)."""
    m = (lambda v: v.abs()) if absolute else (lambda v: v)
    p = {k: v.double() for k, v in p.items()}
    B, T, D = p["u"].shape
    N = p["a_log"].shape[1]
    b, c = (v[:, :, None] if v.dim() == 3 else v for v in (p["b"], p["c"]))
    G = b.shape[2]
    ends = n if n is not None else torch.full((B,), T, device=dy.device)
    on = (torch.arange(T, device=dy.device)[None, :] < ends[:, None])[..., None].double()
    raw = p["dt"] + p["dt_bias"]
    s = torch.logaddexp(raw, torch.zeros_like(raw)) * on
    A = -torch.exp(p["a_log"])
    sz = torch.sigmoid(p["z"])
    dy = m(dy.double()) * on
    q = dy * m(p["z"]) * sz
    wide = lambda v: m(v).repeat_interleave(D // G, 1)  # [B, G, N] -> [B, D, N]  # noqa: E731
    group = lambda v: v.reshape(B, G, D // G, N).sum(2)  # noqa: E731
    su = m(s * p["u"])
    hs = torch.zeros(T + 1, B, D, N, dtype=torch.float64, device=dy.device)
    off = torch.zeros_like(hs) if absolute else None
    step, lost = 2.0 ** -23, lambda x: 2.0 ** -22 - 2.0 ** -21 * x
    for t in range(T):
        x = s[:, t, :, None] * A
        hs[t + 1] = torch.exp(x) * hs[t] + su[:, t, :, None] * wide(b[:, t])
        if absolute:
            off[t + 1] = torch.exp(x) * (off[t] + hs[t] * lost(x)) + step * hs[t + 1]
    got = {k: torch.zeros_like(v) for k, v in p.items()}
    gb, gc = got["b"].view(b.shape), got["c"].view(c.shape)
    pre, v, through_a = (torch.zeros_like(s) for _ in range(3))
    carry = torch.zeros_like(hs[0])
    err = {k: torch.zeros_like(v) for k, v in p.items()}
    eb, ec = err["b"].view(b.shape), err["c"].view(c.shape)
    epre, ev, ethrough_a, ecarry = (torch.zeros_like(w) for w in (s, s, s, carry))
    for t in range(T - 1, -1, -1):
        wb, wc, qt, sut, st = wide(b[:, t]), wide(c[:, t]), q[:, t, :, None], su[:, t, :, None], s[:, t, :, None]
        g, x = wc * qt + carry, st * A
        a = torch.exp(x)
        gc[:, t], gb[:, t] = group(hs[t + 1] * qt), group(g * sut)
        pre[:, t], v[:, t] = (hs[t + 1] * wc).sum(-1), (g * wb).sum(-1)
        carry = g * a
        through = carry * hs[t]
        through_a[:, t] = (through * m(A)).sum(-1)
        got["a_log"] += (through * st).sum(0) * m(A)
        if absolute:
            eg = ecarry + step * g
            ec[:, t], eb[:, t] = group(off[t + 1] * qt), group(eg * sut)
            epre[:, t], ev[:, t] = (off[t + 1] * wc).sum(-1), (eg * wb).sum(-1)
            ecarry = a * (eg + g * lost(x))
            e = ecarry * hs[t] + carry * off[t]
            ethrough_a[:, t] = (e * m(A)).sum(-1)
            err["a_log"] += (e * st).sum(0) * m(A)

    def close(out, pre, v, through_a, extra):
        u, skip = m(p["u"]), m(p["skip"]) * extra
        out["u"] = (v * s + q * skip) * on
        out["dt"] = (through_a + v * u) * torch.sigmoid(raw) * on
        out["z"] = dy * (pre + skip * u) * sz * (1 + m(p["z"]) * (1 - sz))
        out["skip"], out["dt_bias"] = (q * u).sum((0, 1)) * extra, out["dt"].sum((0, 1))
        return out

    got = close(got, pre, v, through_a, 1.0)
    return got, close(err, epre, ev, ethrough_a, 0.0) if absolute else None


@pytest.mark.parametrize("G", [1, 3])
def test_wide_reference(G):
    p, dy, _, n = scan_inputs(3, 14, 12, 5, G, torch.float32, "cpu", 4, lengths=True)
    for a in (False, True):
        want, (got, err) = scan_ref(p, dy, None, n, absolute=a)[2], scan_ref_wide(p, dy, n, absolute=a)
        for k in got:
            assert bool(((got[k] - want[k]).abs() <= 1e-12 * (1 + want[k].abs())).all()), k
            assert not a or bool((err[k] <= 2.0 ** -12 * got[k]).all())


def wide_check(p, dy, n, saved):
    """Gradients against scan_ref_wide: what rounded decays and running sums move, 24
    other roundings and sigmoids of 2^-17, the terms of the longest sum (states of a
    row; channels for b and c; tokens for the parameters, whose sums over sequences
    are in 64 bits), and the rounding to the type."""
    grads = run_scan_bwd(p, dy, saved, lengths=n)
    want, _ = scan_ref_wide(p, dy, n)
    mag, err = scan_ref_wide(p, dy, n, absolute=True)
    B, T, D = dy.shape
    N = p["a_log"].shape[1]
    terms = {"b": N + D, "c": N + D, "a_log": N + T, "skip": N + T, "dt_bias": N + T}
    for k in want:
        got = getattr(grads, "d" + k)
        off = (got.double() - want[k]).abs()
        lim = err[k] + (2.0 ** -17 + (24 + terms.get(k, N)) * 2.0 ** -24) * mag[k]
        lim += HALF[got.dtype] * (want[k].abs() + lim) + 1e-30
        assert bool((off <= lim).all()), f"{k}: off by {float((off / lim).max()):.3g} of the limit"
        del off, lim


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_gradients_by_the_wide_reference(device, dtype):
    p, dy, _, n = scan_inputs(5, 70, 40, 33, 2, dtype, device, 3, lengths=True)
    wide_check(p, dy, n, run_scan(p, lengths=n, save=True)[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N,G", [
    (4, 8300, 520, 33, 1),    # some spans of all sequences at a time, one piece
    (4, 8300, 522, 36, 2),    # the same, groups and rows that are no whole fours
    (1, 10700, 1576, 64, 1),  # the same, in pieces
    (4000, 9, 264, 64, 1),    # some sequences at a time
    (170, 400, 1023, 20, 1),  # the same, fewer states
])
def test_scan_gradients_in_parts(dtype, B, T, D, N, G):
    """Sums by tile past the room that a backward pass takes: it goes part by part,
    with the gradients of the formula, and with no more memory than its outputs,
    the kept states or 1 GB, and a quarter of that for the parameters' sums."""
    p, dy, _, _ = scan_inputs(B, T, D, N, G, dtype, "cuda", B + T)
    p["dt_bias"] -= 1.0
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(7)).to(torch.int32).cuda()
    n[0] = T
    saved = run_scan(p, lengths=n, save=True)[2]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grads = run_scan_bwd(p, dy, saved, lengths=n)
    torch.cuda.synchronize()
    taken = torch.cuda.max_memory_allocated() - before
    outputs = sum(v.numel() * v.element_size() for v in grads)
    del grads
    assert taken <= outputs + 1.25 * max(1 << 30, saved.numel() * 4)
    wide_check(p, dy, n, saved)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [601, 602, 603, 604])
@pytest.mark.parametrize("D,N,G", [(256, 3, 1), (250, 3, 2), (256, 8, 1), (256, 4, 2), (128, 12, 1), (128, 16, 1), (129, 16, 3), (65, 20, 1), (64, 32, 2),
                                   (40, 33, 1), (33, 64, 1), (40, 64, 5)])
def test_single_tokens_of_many_sequences(device, dtype, B, D, N, G):
    """Batches that give a thread four sequences, with one to four in the last
    thread: every lane's share of a channel's states."""
    p, _, state, _ = scan_inputs(B, 1, D, N, G, dtype, device, B + D + N)
    gate = B % 2 == 0
    one = {k: v[:, 0] if k in ("u", "dt", "z", "b", "c") else v for k, v in p.items()}
    if not gate:
        one["z"] = one["dt_bias"] = one["skip"] = None
    q = {k: v.cpu().double() if v is not None else None for k, v in one.items()}
    raw = q["dt"] + (q["dt_bias"] if gate else 0.0)
    s = torch.logaddexp(raw, torch.zeros_like(raw))[..., None]
    A = -torch.exp(q["a_log"])
    wide = lambda v: (v if G == 1 else v.repeat_interleave(D // G, 1)).reshape(B, -1, N)  # noqa: E731
    own, b, c, u = torch.exp(s * A) * state.cpu().double(), wide(q["b"]), wide(q["c"]), q["u"][..., None]
    values = []
    for m in (lambda v: v, lambda v: v.abs()):
        h = m(own) + m(s * u * b)
        y = (m(h) * m(c)).sum(-1) + (m(q["skip"] * q["u"]) if gate else 0.0)
        values.append((y * m(q["z"]) * torch.sigmoid(q["z"]) if gate else y, h))
    (y, h), (my, mh) = values
    rel = limits(p, float((s * -A).max()))[0]
    args = [one[k] for k in ("u", "dt", "a_log", "b", "c")]
    rest = dict(skip=one["skip"], z=one["z"], dt_bias=one["dt_bias"])
    other = torch.full_like(state, 7.0)
    near(ssm.state_scan_step(*args, state, **rest, out_state=other), y, my, rel, "y")
    near(other, h, mh, rel, "state")
    moved = state.clone()
    near(ssm.state_scan_step(*args, moved, **rest), y, my, rel, "y in place")
    assert torch.equal(moved, other)
    # as a piece of one token of a padded batch: sequences of no tokens keep their states
    n = (torch.arange(B, device=device) % 5 != 2).to(torch.int32)
    p = dict(p, skip=rest["skip"], z=p["z"] if gate else None, dt_bias=rest["dt_bias"])
    gy, gh, saved = run_scan(p, state=state, lengths=n, want_state=True, save=True)
    on = n.cpu().bool()
    near(gy[:, 0].cpu()[on], y[on], my[on], rel, "padded y")
    near(gh.cpu()[on], h[on], mh[on], rel, "padded state")
    assert not gy.cpu()[~on].any() and torch.equal(gh.cpu()[~on], state.cpu()[~on]) and torch.equal(saved[:, 0], state)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N,G", [(1, 530, 12, 33, 1), (1, 545, 16, 64, 1), (2, 400, 24, 64, 3), (1, 450, 9, 36, 3),
                                       (3, 420, 20, 20, 2), (1, 700, 130, 8, 1), (2, 610, 66, 5, 2)])
def test_scan_in_pieces_with_many_states_and_groups(device, dtype, B, T, D, N, G):
    """Outputs, states and gradients of calls that are cut along the tokens,
    within what rounded decays move (far less than the sizes of the values)."""
    p, dy, state, _ = scan_inputs(B, T, D, N, G, dtype, device, T + N)
    p["dt_bias"] -= 1.0
    for n in (None, torch.tensor([T, 0, T // 3][:B], dtype=torch.int32, device=device)):
        y, last, saved = run_scan(p, lengths=n, want_state=True, save=True)
        wide_check(p, dy, n, saved)
        forward_check(p, None, n, y, last)
        s = state.clone()
        y, last, _ = run_scan(p, state=s, lengths=n, out_state=s)
        forward_check(p, state, n, y, s)
        if n is not None:
            gone = torch.arange(T, device=device)[None, :] >= n[:, None]
            assert not y[gone].any()


def forward_check(p, state, n, y, last):
    """y and the last state against the formula in 64 bits, as wide_check."""
    B, T, D = y.shape
    N = p["a_log"].shape[1]
    q = {k: v.double() for k, v in p.items()}
    b, c = (v if v.dim() == 4 else v[:, :, None] for v in (q["b"], q["c"]))
    wide = lambda v: v.repeat_interleave(D // v.shape[1], 1)  # noqa: E731
    raw = q["dt"] + q["dt_bias"]
    s, A = torch.logaddexp(raw, torch.zeros_like(raw)), -torch.exp(q["a_log"])
    h = state.double() if state is not None else torch.zeros(B, D, N, dtype=torch.float64, device=y.device)
    mh, eh = h.abs(), torch.zeros_like(h)
    gate = q["z"] * torch.sigmoid(q["z"])
    rest = 2.0 ** -17 + (24 + N) * 2.0 ** -24
    ends = n if n is not None else torch.full((B,), T, device=y.device)
    for t in range(T):
        on = (t < ends)[:, None]
        x = s[:, t, :, None] * A
        own, u, sb = torch.exp(x), q["u"][:, t], (s[:, t] * q["u"][:, t])[..., None] * wide(b[:, t])
        to = own * h + sb, own * mh + sb.abs(), own * (eh + mh * (2.0 ** -22 - 2.0 ** -21 * x))
        h, mh = (torch.where(on[..., None], a, v) for a, v in zip(to, (h, mh)))
        eh = torch.where(on[..., None], to[2] + 2.0 ** -23 * mh, eh)
        wc = wide(c[:, t])
        want = ((h * wc).sum(-1) + q["skip"] * u) * gate[:, t] * on
        mag = ((mh * wc.abs()).sum(-1) + (q["skip"] * u).abs()) * gate[:, t].abs() * on
        lim = (eh * wc.abs()).sum(-1) * gate[:, t].abs() + rest * mag
        lim += HALF[y.dtype] * (want.abs() + lim) + 1e-30
        assert bool(((y[:, t].double() - want).abs() <= lim).all()), t
    assert bool(((last.double() - h).abs() <= eh + rest * mh + 1e-30).all())
