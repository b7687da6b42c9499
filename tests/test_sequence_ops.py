"""The short causal convolution and the selective state space scan: forward,
states, single tokens and gradients against the formulas in 64 bits.

Tolerances.  Every output is a sum of products; `absolute` evaluates the same
formula with every factor's magnitude, so a relative error r of each product
moves the output by at most r times that.  A product's factors are
 - decays, at most 2 T of them in one product: 2^-22 each for the exponential's
   approximation and 2^-21 x for that of its argument x (softplus, product, scaling);
 - at most 24 other roundings of 2^-24, and gates and slopes (sigmoids of
   arguments up to 16, whose exponential is good to 2^-18);
 - the sums' own roundings, 2^-24 for each term of the longest sum.
On top of that comes the rounding to the output's type, half a step of it.
"""
import math

import pytest
import torch

from dlvk_b200.ops import ssm

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def near(got, ref, mag, rel, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got.detach().cpu().double() - ref).abs()
    lim = rel * mag + HALF[got.dtype] * (ref.abs() + rel * mag) + 1e-30
    assert bool((off <= lim).all()), f"{what}: off by {(off / lim).max():.3g} of the limit"


# ------------------------------------------------------------------ convolution
def conv_ref(x, w, bias, state, lengths, silu, dy=None, absolute=False):
    """(y, last state, dx, dw, db) in 64 bits, token by token."""
    m = (lambda v: v.abs()) if absolute else (lambda v: v)
    x, w = x.cpu().double(), w.cpu().double()
    B, T, D = x.shape
    K = w.shape[1]
    n = lengths.tolist() if lengths is not None else [T] * B
    bias = bias.cpu().double() if bias is not None else torch.zeros(D, dtype=torch.float64)
    state = state.cpu().double() if state is not None else torch.zeros(B, K - 1, D, dtype=torch.float64)
    y, dx = torch.zeros(B, T, D, dtype=torch.float64), torch.zeros(B, T, D, dtype=torch.float64)
    dw, db, last = torch.zeros_like(w), torch.zeros_like(bias), torch.zeros_like(state)
    for i in range(B):
        seq = torch.cat([state[i], x[i, :n[i]]])
        last[i] = seq[n[i]:]
        for t in range(n[i]):
            win = seq[t:t + K]  # [K, D]
            p = (win * w.t()).sum(0) + bias
            big = (m(win) * m(w.t())).sum(0) + m(bias)  # the sum's size
            s = torch.sigmoid(p)
            y[i, t] = (big if absolute else p) * (s if silu else 1)
            if silu and absolute:  # the slope of silu is at most 1.1, so p's error reaches y 1.1 times
                y[i, t] = 1.1 * big
            if dy is not None:
                g = m(dy[i, t].cpu().double())
                slope = s * (1 + p * (1 - s))
                if silu:  # second derivative at most 0.5: the error of p
                    g = g * (s * (1 + p.abs() * (1 - s)) + 0.5 * big if absolute else slope)
                db += g
                dw += (m(win) * g).t()
                for j in range(K):
                    if t - K + 1 + j >= 0:
                        dx[i, t - K + 1 + j] += m(w[:, j]) * g
    return y, last, dx, dw, db


def conv_inputs(B, T, D, K, dtype, device, seed=0, lengths=False):
    g = gen(seed)
    x = torch.randn(B, T, D, generator=g).to(dtype).to(device)
    dy = torch.randn(B, T, D, generator=g).to(dtype).to(device)
    w = (torch.randn(D, K, generator=g) * 0.5).to(device)
    b = torch.randn(D, generator=g).to(device)
    s = torch.randn(B, K - 1, D, generator=g).to(dtype).to(device)
    n = None
    if lengths:
        n = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32)
        n[0] = 0
        n = n.to(device)
    return x, dy, w, b, s, n


def conv_check(x, dy, w, b, s, n, silu):
    ref, mag = (conv_ref(x, w, b, s, n, silu, dy, absolute=a) for a in (False, True))
    y, last = ssm.short_conv_fwd(x, w, b, state=s, lengths=n, silu=silu, want_state=True)
    assert y.dtype == x.dtype and last.dtype == x.dtype
    rel = 2.0 ** -18
    near(y, ref[0], mag[0], rel, "y")
    assert torch.equal(last.cpu().double(), ref[1])
    y2, none = ssm.short_conv_fwd(x, w, b, state=s, lengths=n, silu=silu)
    assert none is None and torch.equal(y, y2)
    dx, dw, db = ssm.short_conv_bwd(x, w, b, dy, state=s, lengths=n, silu=silu)
    assert dw.dtype == torch.float32 and (db is None) == (b is None)
    terms = x.shape[0] * x.shape[1] * 2.0 ** -24
    near(dx, ref[2], mag[2], rel, "dx")
    near(dw, ref[3], mag[3], rel + terms, "dw")
    if b is not None:
        near(db, ref[4], mag[4], rel + terms, "db")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,K", [(1, 1, 1, 4), (2, 1, 64, 4), (3, 2, 40, 3), (1, 15, 8, 2), (2, 16, 257, 4),
                                     (2, 17, 264, 4), (1, 50, 33, 3), (9, 5, 24, 2), (4, 33, 520, 4)])
def test_conv(device, dtype, B, T, D, K):
    x, dy, w, b, s, n = conv_inputs(B, T, D, K, dtype, device, B + T + D)
    conv_check(x, dy, w, b, s, None, True)
    conv_check(x, dy, w, None, None, None, False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 3, 16, 40])
@pytest.mark.parametrize("K", [2, 4])
def test_conv_lengths_and_what_lies_behind_them(device, dtype, T, K):
    x, dy, w, b, s, n = conv_inputs(6, T, 48, K, dtype, device, T, lengths=True)
    conv_check(x, dy, w, b, s, n, True)
    gone = (torch.arange(T, device=device)[None, :] >= n[:, None])[..., None].expand_as(x)
    xn = torch.where(gone, torch.full_like(x, math.nan), x)
    dyn = torch.where(gone, torch.full_like(x, math.inf), dy)
    for a, c in zip(ssm.short_conv_fwd(x, w, b, state=s, lengths=n, want_state=True),
                    ssm.short_conv_fwd(xn, w, b, state=s, lengths=n, want_state=True)):
        assert torch.equal(a, c)
    for a, c in zip(ssm.short_conv_bwd(x, w, b, dy, state=s, lengths=n),
                    ssm.short_conv_bwd(xn, w, b, dyn, state=s, lengths=n)):
        assert torch.equal(a, c)
    assert not ssm.short_conv_fwd(xn, w, b, lengths=n)[0][gone].any()
    # lengths outside [0, T] are taken as its ends
    m = torch.tensor([-3, 0, T, T + 5, T, T], dtype=torch.int32, device=device)
    a = ssm.short_conv_fwd(x, w, b, state=s, lengths=m, want_state=True)
    c = ssm.short_conv_fwd(x, w, b, state=s, lengths=m.clamp(0, T), want_state=True)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_conv_views_and_given_outputs(device, dtype):
    x, dy, w, b, s, _ = conv_inputs(3, 21, 32, 4, dtype, device, 5)
    want = ssm.short_conv_bwd(x, w, b, dy, state=s)
    wy, ws = ssm.short_conv_fwd(x, w, b, state=s, want_state=True)
    for off, width in ((0, 64), (8, 72), (3, 67)):
        base = torch.full((3, 21, width), 7.0, device=device, dtype=dtype)
        xv = base[:, :, off:off + 32]
        xv.copy_(x)
        y, last = ssm.short_conv_fwd(xv, w, b, state=s, want_state=True)
        assert torch.equal(y, wy) and torch.equal(last, ws)
        out = torch.full((3, 21, width), 7.0, device=device, dtype=dtype)
        got = ssm.short_conv_bwd(xv, w, b, dy, state=s, dx=out[:, :, off:off + 32])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert bool((out[:, :, :off] == 7).all()) and bool((out[:, :, off + 32:] == 7).all())
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(ssm.short_conv_fwd(turned, w, b, state=s)[0], wy)
    dw, db = torch.ones_like(w), torch.ones_like(b)
    ssm.short_conv_bwd(x, w, b, dy, state=s, dweight=dw, dbias=db, accumulate=True)
    assert bool(((dw - 1 - want[1]).abs() <= 2.0 ** -23 * (1 + want[1].abs())).all())
    assert bool(((db - 1 - want[2]).abs() <= 2.0 ** -23 * (1 + want[2].abs())).all())
    ones = dy[:1, :1].expand(3, 21, 32)
    assert torch.equal(ssm.short_conv_bwd(x, w, b, ones, state=s)[0], ssm.short_conv_bwd(x, w, b, ones.contiguous(), state=s)[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [5, 64])
def test_conv_pieces_and_single_tokens(device, dtype, D):
    x, _, w, b, s, _ = conv_inputs(2, 23, D, 4, dtype, device, D)
    y, last = ssm.short_conv_fwd(x, w, b, state=s, want_state=True)
    ref, mag = (conv_ref(x, w, b, s, None, True, absolute=a)[0] for a in (False, True))

    def same(got, t0, t1):
        if device == "cuda":  # the kernel's bits do not depend on the pieces
            assert torch.equal(got, y[:, t0:t1])
        # torch's vector and remainder loops on the CPU differ in the last bits of a sigmoid
        near(got, ref[:, t0:t1], mag[:, t0:t1], 2.0 ** -18, "piece")

    state, parts = s.clone(), []
    for a, e in ((0, 1), (1, 3), (3, 19), (19, 19), (19, 23)):  # the state moves on in place
        parts.append(ssm.short_conv_fwd(x[:, a:e], w, b, state=state, out_state=state)[0])
    same(torch.cat(parts, 1), 0, 23)
    assert torch.equal(state, last)
    state = s.clone()
    for t in range(23):
        same(ssm.short_conv_step(x[:, t], w, b, state)[:, None], t, t + 1)
    assert torch.equal(state, last)
    other = torch.empty_like(s)
    keep = s.clone()
    same(ssm.short_conv_step(x[:, 0], w, b, s, out_state=other)[:, None], 0, 1)
    assert torch.equal(s, keep) and torch.equal(other, torch.cat([s[:, 1:], x[:, :1]], 1))


@pytest.mark.parametrize("device", DEVICES)
def test_conv_empty(device):
    x, dy, w, b, s, _ = conv_inputs(2, 4, 8, 4, torch.float32, device)
    y, last = ssm.short_conv_fwd(x[:, :0], w, b, state=s, want_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(last, s)
    assert not ssm.short_conv_fwd(x[:, :0], w, b, want_state=True)[1].any()
    assert ssm.short_conv_fwd(x[:0], w, b)[0].shape == (0, 4, 8)
    for part in (x[:, :0], x[:0]):
        dx, dw, db = ssm.short_conv_bwd(part, w, b, part)
        assert dx.shape == part.shape and not dw.any() and not db.any()


@pytest.mark.parametrize("device", DEVICES)
def test_conv_refusals(device):
    x, dy, w, b, s, n = conv_inputs(2, 6, 8, 4, torch.float32, device, lengths=True)
    bad = (ValueError, RuntimeError)
    for call in (lambda: ssm.short_conv_fwd(x.half(), w, b), lambda: ssm.short_conv_fwd(x[0], w, b),
                 lambda: ssm.short_conv_fwd(x, w[:, :1], b), lambda: ssm.short_conv_fwd(x, torch.ones(8, 5, device=device), b),
                 lambda: ssm.short_conv_fwd(x, w[:7], b), lambda: ssm.short_conv_fwd(x, w.bfloat16(), b),
                 lambda: ssm.short_conv_fwd(x, w, b[:3]), lambda: ssm.short_conv_fwd(x, w, b, state=s[:, :2]),
                 lambda: ssm.short_conv_fwd(x, w, b, state=s.bfloat16()), lambda: ssm.short_conv_fwd(x, w, b, lengths=n.long()),
                 lambda: ssm.short_conv_fwd(x, w, b, lengths=n[:1]), lambda: ssm.short_conv_fwd(x, w, b, out_state=s[:, :1]),
                 lambda: ssm.short_conv_bwd(x, w, b, dy[:, :5]), lambda: ssm.short_conv_bwd(x, w, b, dy.bfloat16()),
                 lambda: ssm.short_conv_bwd(x, w, b, dy, accumulate=True),
                 lambda: ssm.short_conv_bwd(x, w, None, dy, dbias=torch.zeros(8, device=device)),
                 lambda: ssm.short_conv_bwd(x, w, b, dy, dweight=torch.zeros(4, 8, device=device))):
        with pytest.raises(bad):
            call()


@pytest.mark.gpu
def test_conv_refusals_of_memory():
    x, dy, w, b, s, _ = conv_inputs(2, 6, 8, 4, torch.float32, "cuda")
    for call in (lambda: ssm.short_conv_bwd(x, w, b, dy, dx=x), lambda: ssm.short_conv_bwd(x, w, b, dy, dx=dy),
                 lambda: ssm.short_conv_bwd(x, w, b, dy, dx=x[:1].expand(2, 6, 8)),
                 lambda: ssm.short_conv_fwd(x, w.cpu(), b), lambda: ssm.short_conv_fwd(x, w, b, state=s.cpu()),
                 lambda: ssm.short_conv_bwd(x, w, b, dy, dweight=w),
                 lambda: ssm.short_conv_fwd(x[:, :3], w, b, out_state=x[:, :3]),
                 lambda: ssm.short_conv_fwd(x[:, :4], w, b, state=x[:, :3], out_state=x[:, 3:]),
                 lambda: ssm.short_conv_fwd(x[:, 5:], w, b, state=x[:, :3], out_state=x[:, 1:4]),
                 lambda: ssm.short_conv_bwd(x, w, b, dy, dx=torch.empty(2, 8, 6, device="cuda").transpose(1, 2))):
        with pytest.raises(RuntimeError):
            call()


# ------------------------------------------------------------------------- scan
NAMES = ("u", "dt", "a_log", "b", "c", "skip", "z", "dt_bias")


def scan_inputs(B, T, D, N, G, dtype, device, seed=0, full=True, lengths=False):
    g = gen(seed)
    rows = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    p = {"u": rows(B, T, D), "dt": rows(B, T, D), "b": rows(B, T, G, N) if G > 1 else rows(B, T, N)}
    p["c"] = torch.randn(p["b"].shape, generator=g).to(dtype).to(device)
    p["a_log"] = (torch.randn(D, N, generator=g) * 0.7).to(device)
    p["skip"], p["dt_bias"], p["z"] = None, None, None
    if full:
        p["skip"] = torch.randn(D, generator=g).to(device)
        p["dt_bias"] = (torch.randn(D, generator=g) - 2.0).to(device)
        p["z"] = rows(B, T, D)
    dy = rows(B, T, D)
    state = torch.randn(B, D, N, generator=g).to(device)
    n = None
    if lengths:
        n = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32)
        n[0] = 0
        n = n.to(device)
    return p, dy, state, n


def scan_ref(p, dy, state, n, absolute=False):
    """y, last state and gradients in 64 bits, by the formulas; with `absolute`
    the magnitudes of all products."""
    m = (lambda v: v.abs()) if absolute else (lambda v: v)
    p = {k: v.cpu().double() if v is not None else None for k, v in p.items()}
    u, dt, b, c = p["u"], p["dt"], p["b"], p["c"]
    B, T, D = u.shape
    N = p["a_log"].shape[1]
    if b.dim() == 3:
        b, c = b[:, :, None], c[:, :, None]
    G = b.shape[2]
    zero = torch.zeros(D, dtype=torch.float64)
    skip = p["skip"] if p["skip"] is not None else zero
    bias = p["dt_bias"] if p["dt_bias"] is not None else zero
    A = -torch.exp(p["a_log"])
    dy = dy.cpu().double() if dy is not None else torch.zeros_like(u)
    n = n.cpu().clamp(0, T).tolist() if n is not None else [T] * B
    got = {k: torch.zeros_like(v) for k, v in (("u", u), ("dt", dt), ("a_log", A), ("b", b), ("c", c), ("skip", zero),
                                               ("z", u), ("dt_bias", zero))}
    y, last = torch.zeros_like(u), torch.zeros(B, D, N, dtype=torch.float64)
    wide = lambda v: v.repeat_interleave(D // G, 0)  # [G, N] -> [D, N]  # noqa: E731
    group = lambda v: v.reshape(G, D // G, N).sum(1)  # noqa: E731
    xmax = 0.0
    for i in range(B):
        h = m(state[i].cpu().double()) if state is not None else torch.zeros(D, N, dtype=torch.float64)
        hs, decays = [h], []
        for t in range(n[i]):
            s = torch.logaddexp(dt[i, t] + bias, zero)
            decays.append(torch.exp(s[:, None] * A))
            xmax = max(xmax, float((s[:, None] * -A).max()))
            h = decays[-1] * h + m(s * u[i, t])[:, None] * m(wide(b[i, t]))
            hs.append(h)
            pre = (h * m(wide(c[i, t]))).sum(1) + m(skip * u[i, t])
            z = p["z"][i, t] if p["z"] is not None else None
            y[i, t] = pre * (m(z) * torch.sigmoid(z) if z is not None else 1)
        last[i] = h
        carry = torch.zeros(D, N, dtype=torch.float64)
        for t in range(n[i] - 1, -1, -1):
            raw = dt[i, t] + bias
            s, z = torch.logaddexp(raw, zero), p["z"][i, t] if p["z"] is not None else None
            q = m(dy[i, t])
            if z is not None:
                sz = torch.sigmoid(z)
                pre = (hs[t + 1] * m(wide(c[i, t]))).sum(1) + m(skip * u[i, t])
                got["z"][i, t] = q * pre * sz * (1 + m(z) * (1 - sz))
                q = q * m(z) * sz
            g = m(wide(c[i, t])) * q[:, None] + carry
            got["c"][i, t] = group(hs[t + 1] * q[:, None])
            got["b"][i, t] = group(g * m(s * u[i, t])[:, None])
            v = (g * m(wide(b[i, t]))).sum(1)
            carry = g * decays[t]
            through = carry * hs[t]
            got["u"][i, t] = v * s + q * m(skip)
            d = ((through * m(A)).sum(1) + v * m(u[i, t])) * torch.sigmoid(raw)
            got["dt"][i, t] = d
            got["dt_bias"] += d
            got["skip"] += q * m(u[i, t])
            got["a_log"] += through * m(A) * s[:, None]
    got["b"], got["c"] = got["b"].reshape(p["b"].shape), got["c"].reshape(p["c"].shape)
    return y, last, got, xmax


def run_scan(p, **kw):
    return ssm.state_scan_fwd(p["u"], p["dt"], p["a_log"], p["b"], p["c"], p["skip"], p["z"], p["dt_bias"], **kw)


def run_scan_bwd(p, dy, saved, **kw):
    return ssm.state_scan_bwd(p["u"], p["dt"], p["a_log"], p["b"], p["c"], dy, saved, p["skip"], p["z"], p["dt_bias"], **kw)


def limits(p, xmax):
    B, T, D = p["u"].shape
    N = p["a_log"].shape[1]
    own = 2 * T * (2.0 ** -22 + xmax * 2.0 ** -21) + 24 * 2.0 ** -24 + 2.0 ** -17
    return own + (N + 2) * 2.0 ** -24, own + (N + D + B * T) * 2.0 ** -24


def scan_check(p, dy, state, n):
    (y, last, g, xmax), (my, ml, mg, _) = scan_ref(p, dy, state, n), scan_ref(p, dy, state, n, absolute=True)
    short, long = limits(p, xmax)
    gy, gl, saved = run_scan(p, state=state, lengths=n, want_state=True, save=True)
    assert gy.dtype == p["u"].dtype and gl.dtype == torch.float32
    near(gy, y, my, short, "y")
    near(gl, last, ml, short, "state")
    y2, l2, s2 = run_scan(p, state=state, lengths=n)
    assert l2 is None and s2 is None and torch.equal(y2, gy)
    grads = run_scan_bwd(p, dy, saved, lengths=n)
    for k, name in (("du", "u"), ("ddt", "dt"), ("da_log", "a_log"), ("db", "b"), ("dc", "c"), ("dskip", "skip"),
                    ("dz", "z"), ("ddt_bias", "dt_bias")):
        got = getattr(grads, k)
        if p[name] is None:
            assert got is None
            continue
        assert got.dtype == p[name].dtype
        near(got, g[name], mg[name], long, k)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N,G", [(1, 1, 1, 1, 1), (2, 1, 40, 16, 1), (1, 3, 8, 4, 1), (2, 15, 33, 5, 1), (1, 16, 64, 8, 2),
                                       (3, 17, 24, 16, 3), (1, 34, 72, 17, 1), (2, 20, 16, 33, 2), (1, 18, 20, 64, 1),
                                       (1, 70, 130, 9, 1), (2, 33, 264, 16, 1)])
def test_scan(device, dtype, B, T, D, N, G):
    p, dy, state, _ = scan_inputs(B, T, D, N, G, dtype, device, B + T + D + N)
    scan_check(p, dy, state, None)
    p, dy, _, _ = scan_inputs(B, T, D, N, G, dtype, device, B + T, full=False)
    scan_check(p, dy, None, None)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N", [(1, 257, 8, 16), (2, 300, 12, 3), (1, 530, 7, 20)])
def test_scan_of_many_tokens(device, dtype, B, T, D, N):
    """Long enough to be cut into pieces; states that last across them."""
    p, dy, state, n = scan_inputs(B, T, D, N, 1, dtype, device, T, lengths=B > 1)
    p["dt_bias"] -= 3.0
    p["a_log"] -= 2.0
    scan_check(p, dy, state, n)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N", [(1, 16), (5, 4), (16, 16), (41, 16), (37, 64)])
def test_scan_lengths_and_what_lies_behind_them(device, dtype, T, N):
    p, dy, state, n = scan_inputs(5, T, 24, N, 1, dtype, device, T, lengths=True)
    scan_check(p, dy, state, n)
    gone = (torch.arange(T, device=device)[None, :] >= n[:, None])[..., None]
    bad = dict(p)
    for k, v in (("u", math.nan), ("dt", math.inf), ("z", -math.inf), ("b", math.nan), ("c", math.inf)):
        bad[k] = torch.where(gone.expand_as(p[k]), torch.full_like(p[k], v), p[k])
    bad_dy = torch.where(gone.expand_as(dy), torch.full_like(dy, math.nan), dy)
    a = run_scan(p, state=state, lengths=n, want_state=True, save=True)
    c = run_scan(bad, state=state, lengths=n, want_state=True, save=True)
    assert all(torch.equal(i, j) for i, j in zip(a, c))
    assert not c[0][gone.expand_as(dy)].any()
    assert torch.equal(c[1][0], state[0])  # the empty sequence's
    ga, gc = run_scan_bwd(p, dy, a[2], lengths=n), run_scan_bwd(bad, bad_dy, c[2], lengths=n)
    for i, j in zip(ga, gc):
        assert torch.equal(i, j)
    for k in ("du", "ddt", "dz", "db", "dc"):
        v = getattr(gc, k)
        assert not v[gone.expand_as(v)].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_views_and_given_outputs(device, dtype):
    p, dy, state, _ = scan_inputs(2, 19, 40, 16, 1, dtype, device, 11)
    y, last, saved = run_scan(p, state=state, want_state=True, save=True)
    want = run_scan_bwd(p, dy, saved)
    mag = scan_ref(p, dy, state, None, absolute=True)[2]
    for off in (0, 8, 3):
        wide = torch.full((2, 19, 3 * 40 + 2 * 16 + off), 5.0, device=device, dtype=dtype)
        q, at = dict(p), off
        for k in ("u", "dt", "z", "b", "c"):
            q[k] = wide[:, :, at:at + p[k].shape[2]]
            q[k].copy_(p[k])
            at += p[k].shape[2]
        got = run_scan(q, state=state, want_state=True, save=True)
        assert all(torch.equal(a, b) for a, b in zip(got, (y, last, saved)))
        out, at, given = torch.full_like(wide, 5.0), off, {}
        for k in ("u", "dt", "z", "b", "c"):
            given["d" + k] = out[:, :, at:at + p[k].shape[2]]
            at += p[k].shape[2]
        got = run_scan_bwd(q, dy, saved, **given)
        for k, a in got._asdict().items():
            if k in ("dskip", "ddt_bias"):  # sums over threads, whose channels depend on the alignment
                lim = 2 * (2 * 19) * 2.0 ** -24 * mag[k[1:]]  # B T terms, added in two orders
                assert bool(((a - getattr(want, k)).abs().cpu() <= lim).all())
            else:
                assert torch.equal(a, getattr(want, k))
        assert bool((out[:, :, :off] == 5).all()) and got.du.data_ptr() == given["du"].data_ptr()
    acc = {"da_log": torch.ones_like(p["a_log"]), "dskip": torch.ones(40, device=device),
           "ddt_bias": torch.ones(40, device=device)}
    run_scan_bwd(p, dy, saved, accumulate=True, **acc)
    for k, v in acc.items():
        w = getattr(want, k)
        assert bool(((v - 1 - w).abs() <= 2.0 ** -22 * (1 + w.abs())).all())
    ones = dy[:1, :1].expand_as(dy)  # the gradient of a sum
    for a, b in zip(run_scan_bwd(p, ones, saved), run_scan_bwd(p, ones.contiguous(), saved)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,N,G", [(24, 16, 1), (7, 3, 1), (16, 33, 2)])
def test_scan_pieces_and_single_tokens(device, dtype, D, N, G):
    T = 37
    p, _, state, _ = scan_inputs(2, T, D, N, G, dtype, device, D)
    (y, last, _, xmax), (my, ml, _, _) = scan_ref(p, None, state, None), scan_ref(p, None, state, None, absolute=True)
    rel = limits(p, xmax)[0]
    s, parts = state.clone(), []
    for a, e in ((0, 1), (1, 17), (17, 17), (17, T)):
        piece = {k: v[:, a:e] if k in ("u", "dt", "z", "b", "c") else v for k, v in p.items()}
        parts.append(run_scan(piece, state=s, out_state=s)[0])
    near(torch.cat(parts, 1), y, my, rel, "pieces")
    near(s, last, ml, rel, "state of pieces")
    s = state.clone()
    for t in range(T):
        got = ssm.state_scan_step(p["u"][:, t], p["dt"][:, t], p["a_log"], p["b"][:, t], p["c"][:, t], s, skip=p["skip"],
                                  z=p["z"][:, t], dt_bias=p["dt_bias"])
        near(got, y[:, t], my[:, t], rel, "token")
    near(s, last, ml, rel, "state of tokens")
    other, keep = torch.empty_like(state), state.clone()
    one = ssm.state_scan_step(p["u"][:, 0], p["dt"][:, 0], p["a_log"], p["b"][:, 0], p["c"][:, 0], state, out_state=other)
    assert torch.equal(state, keep) and one.shape == (2, D) and not torch.equal(other, keep)


@pytest.mark.parametrize("device", DEVICES)
def test_scan_empty_and_extreme(device):
    p, dy, state, _ = scan_inputs(2, 4, 8, 4, 1, torch.float32, device)
    none = {k: v[:, :0] if k in ("u", "dt", "z", "b", "c") else v for k, v in p.items()}
    y, last, saved = run_scan(none, state=state, want_state=True, save=True)
    assert y.shape == (2, 0, 8) and torch.equal(last, state)
    g = run_scan_bwd(none, dy[:, :0], saved)
    assert not g.da_log.any() and not g.dskip.any() and not g.ddt_bias.any()
    none = {k: v[:0] if k in ("u", "dt", "z", "b", "c") else v for k, v in p.items()}
    y, last, saved = run_scan(none, want_state=True, save=True)
    assert y.shape == (0, 4, 8) and last.shape == (0, 8, 4)
    assert not run_scan_bwd(none, dy[:0], saved).da_log.any()
    # steps of no time and of very much: the state stays, or is the last token's alone
    far = dict(p, dt=torch.full_like(p["dt"], -200.0), dt_bias=None)
    assert torch.equal(run_scan(far, state=state, want_state=True)[1], state)
    far = dict(p, dt=torch.full_like(p["dt"], 1000.0), dt_bias=None)
    last = run_scan(far, state=state, want_state=True)[1]
    ref = 1000.0 * p["u"][:, -1, :, None] * p["b"][:, -1, None, :]
    assert bool(((last - ref).abs() <= 2.0 ** -22 * ref.abs()).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_gradients_against_differences(device, dtype):
    p, dy, _, n = scan_inputs(2, 21, 12, 5, 1, dtype, device, 3, lengths=True)
    _, _, saved = run_scan(p, lengths=n, save=True)
    grads = run_scan_bwd(p, dy, saved, lengths=n)._asdict()

    def value(q):
        return float((scan_ref(q, None, None, n)[0] * dy.cpu().double()).sum())

    g = gen(9)
    mags = scan_ref(p, dy, None, n, absolute=True)[2]
    short, long = limits(p, 4.0)
    for name in NAMES:
        at = p[name].cpu().double()
        v = torch.randn(at.shape, generator=g, dtype=torch.float64)
        step = 1e-4
        q = {k: t.cpu().double() for k, t in p.items()}
        slope = (value(dict(q, **{name: at + step * v})) - value(dict(q, **{name: at - step * v}))) / (2 * step)
        got = grads["d" + name].cpu().double()
        # roundings of the gradient, and differences off by step^2 of third derivatives
        lim = float(((long + HALF[grads["d" + name].dtype]) * mags[name] * v.abs()).sum()) + 1e-5 * float((mags[name] * v.abs()).sum())
        assert abs(float((got * v).sum()) - slope) <= lim, name


@pytest.mark.parametrize("device", DEVICES)
def test_scan_refusals(device):
    p, dy, state, n = scan_inputs(2, 6, 8, 4, 1, torch.float32, device, lengths=True)
    saved = run_scan(p, save=True)[2]
    bad = (ValueError, RuntimeError)
    z = lambda *s: torch.zeros(*s, device=device)  # noqa: E731
    for q in (dict(p, u=p["u"].half()), dict(p, dt=p["dt"].bfloat16()), dict(p, dt=p["dt"][:, :5]),
              dict(p, a_log=z(8, 65)), dict(p, a_log=z(7, 4)), dict(p, a_log=p["a_log"].bfloat16()),
              dict(p, b=p["b"][..., :3]), dict(p, c=p["c"][:1]), dict(p, b=z(2, 6, 3, 4), c=z(2, 6, 3, 4)),
              dict(p, b=z(2, 6, 0, 4), c=z(2, 6, 0, 4)), dict(p, c=z(2, 6, 1, 4)), dict(p, skip=z(7)),
              dict(p, dt_bias=z(8, 1)), dict(p, z=p["z"][:, :, :4]), dict(p, u=p["u"][0])):
        with pytest.raises(bad):
            run_scan(q)
    for kw in (dict(state=state[:, :, :3]), dict(state=state.bfloat16()), dict(lengths=n.long()), dict(lengths=n[:1]),
               dict(out_state=z(2, 8, 5))):
        with pytest.raises(bad):
            run_scan(p, **kw)
    for call in (lambda: run_scan_bwd(p, dy[:, :3], saved), lambda: run_scan_bwd(p, dy, saved[:, :, :4]),
                 lambda: run_scan_bwd(p, dy, saved, accumulate=True), lambda: run_scan_bwd(p, dy, saved, da_log=z(8, 3)),
                 lambda: run_scan_bwd(dict(p, z=None), dy, saved, dz=z(2, 6, 8)),
                 lambda: run_scan_bwd(dict(p, skip=None), dy, saved, dskip=z(8))):
        with pytest.raises(bad):
            call()


@pytest.mark.gpu
def test_scan_refusals_of_memory():
    p, dy, state, _ = scan_inputs(2, 6, 8, 4, 1, torch.float32, "cuda")
    saved = run_scan(p, save=True)[2]
    one = torch.empty(2, 6, 8, device="cuda")
    for call in (lambda: run_scan_bwd(p, dy, saved, du=one, ddt=one), lambda: run_scan_bwd(p, dy, saved, du=p["u"]),
                 lambda: run_scan_bwd(p, dy, saved, dz=dy), lambda: run_scan_bwd(p, dy, saved, du=one[:1].expand(2, 6, 8)),
                 lambda: run_scan_bwd(p, dy, saved, da_log=p["a_log"]), lambda: run_scan(dict(p, z=p["z"].cpu())),
                 lambda: run_scan(p, out_state=torch.empty(2, 4, 8, device="cuda").transpose(1, 2)),
                 lambda: run_scan_bwd(p, dy, saved, du=torch.empty(2, 8, 6, device="cuda").transpose(1, 2))):
        with pytest.raises(RuntimeError):
            call()


# -------------------------------------------------------- streams, graphs, repeats
def everything(p, dy, state, w, bias, cs):
    y, last = ssm.short_conv_fwd(p["u"], w, bias, state=cs, want_state=True)
    out = [y, last, *ssm.short_conv_bwd(p["u"], w, bias, dy, state=cs)]
    y, last, saved = run_scan(p, state=state, want_state=True, save=True)
    return out + [y, last, *run_scan_bwd(p, dy, saved)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_streams_and_graphs(dtype):
    p, dy, state, _ = scan_inputs(3, 45, 136, 16, 1, dtype, "cuda", 21)
    w, bias = torch.randn(136, 4, device="cuda"), torch.randn(136, device="cuda")
    cs = torch.randn(3, 3, 136, device="cuda").to(dtype)
    args = (p, dy, state, w, bias, cs)
    want = everything(*args)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(everything(*args), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs of the same inputs, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = everything(*args)
        graphs.append((g, out))
    p["u"].mul_(0.5)
    want = everything(*args)
    for _ in range(2):
        for g, out in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens_channels_and_sequences(dtype):
    """Sizes where work is cut into pieces: sums of states against the running
    form of the operator itself, token by token in pieces of other sizes."""
    for B, T, D in ((1, 3001, 24), (1, 900, 1048), (70, 40, 33), (2, 2500, 8)):
        p, _, state, _ = scan_inputs(B, T, D, 16, 1, dtype, "cuda", T)
        p["dt_bias"] -= 2.0  # steps short enough for states that last
        y, last, _ = run_scan(p, state=state, want_state=True)
        s, parts = state.clone(), []
        for a in range(0, T, 333):
            piece = {k: v[:, a:a + 333] if k in ("u", "dt", "z", "b", "c") else v for k, v in p.items()}
            parts.append(run_scan(piece, state=s, out_state=s)[0])
        parts = torch.cat(parts, 1)
        # both are within the module's limit of the exact values; states last 1 / (1 - decay) < 400 steps
        size = float(last.abs().max())
        assert float((last - s).abs().max()) <= 2 * 400 * 2.0 ** -20 * size
        off = (y.float() - parts.float()).abs()
        assert bool((off <= (2 * HALF[dtype]) * y.float().abs() + 2 * 400 * 2.0 ** -20 * float(y.float().abs().max())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_states_in_place_in_pieces(dtype):
    """A call that is cut along its tokens and moves its state on in place."""
    p, dy, state, n = scan_inputs(2, 700, 12, 16, 1, dtype, "cuda", 31)
    n = torch.tensor([700, 389], dtype=torch.int32, device="cuda")
    y, last, _ = run_scan(p, state=state, lengths=n, want_state=True)
    s = state.clone()
    y2, same, _ = run_scan(p, state=s, lengths=n, out_state=s)
    assert same.data_ptr() == s.data_ptr() and torch.equal(y2, y) and torch.equal(s, last)
    w = torch.randn(12, 4, device="cuda")
    cs = torch.randn(2, 3, 12, device="cuda").to(dtype)
    y, last = ssm.short_conv_fwd(p["u"], w, state=cs, lengths=n, want_state=True)
    y2, same = ssm.short_conv_fwd(p["u"], w, state=cs, lengths=n, out_state=cs)
    assert same.data_ptr() == cs.data_ptr() and torch.equal(y2, y) and torch.equal(cs, last)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_gradients_in_pieces_with_lengths(device, dtype):
    p, dy, state, _ = scan_inputs(3, 420, 8, 16, 1, dtype, device, 33)
    p["dt_bias"] -= 2.0
    scan_check(p, dy, state, torch.tensor([420, 0, 131], dtype=torch.int32, device=device))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_past_31_bits(dtype):
    """Tokens 2^20 elements apart, in one buffer of 2^32 or so: the same bits as
    from and to dense tensors."""
    T, D, N, apart = 2100, 32, 16, 1 << 20
    buffer = torch.empty(T * apart, dtype=dtype, device="cuda")
    p, dy, _, _ = scan_inputs(1, T, D, N, 1, dtype, "cuda", 35)
    at = [64]

    def spread(t):
        v = buffer.as_strided((1, T, t.shape[-1]), (T * apart, apart, 1), at[0])
        at[0] += 64
        return v.copy_(t) if t is not None else v

    q = {k: spread(v) if k in ("u", "dt", "z", "b", "c") else v for k, v in p.items()}
    far = spread(dy)
    y, last, saved = run_scan(p, want_state=True, save=True)
    y2, last2, saved2 = run_scan(q, want_state=True, save=True)
    assert torch.equal(y, y2) and torch.equal(last, last2) and torch.equal(saved, saved2)
    want = run_scan_bwd(p, dy, saved)
    given = {k: spread(getattr(want, k)) for k in ("du", "ddt", "db", "dc", "dz")}
    for v in given.values():
        v.fill_(7.0)
    got = run_scan_bwd(q, far, saved, **given)
    assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)
    w, bias = torch.randn(D, 4, device="cuda"), torch.randn(D, device="cuda")
    assert torch.equal(ssm.short_conv_fwd(q["u"], w, bias)[0], ssm.short_conv_fwd(p["u"], w, bias)[0])
    given["du"].fill_(7.0)
    want = ssm.short_conv_bwd(p["u"], w, bias, dy)
    assert all(torch.equal(a, b) for a, b in zip(ssm.short_conv_bwd(q["u"], w, bias, far, dx=given["du"]), want))


@pytest.mark.gpu
def test_elements_past_31_bits():
    """70000 sequences of 16 tokens of 2048 channels: the last ones as by themselves."""
    B, T, D, N = 70000, 16, 2048, 16
    g = torch.Generator("cuda").manual_seed(3)
    r = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda").normal_(generator=g)  # noqa: E731
    u, dt, dy, b, c = r(B, T, D), r(B, T, D), r(B, T, D), r(B, T, N), r(B, T, N)
    a_log, skip = torch.rand(D, N, device="cuda"), torch.rand(D, device="cuda")
    some = lambda v: v[-300:].clone()  # noqa: E731
    y, last, saved = ssm.state_scan_fwd(u, dt, a_log, b, c, skip, want_state=True, save=True)
    few = (some(u), some(dt), a_log, some(b), some(c))
    want = ssm.state_scan_fwd(*few, skip, want_state=True, save=True)
    assert all(torch.equal(some(x), w) for x, w in zip((y, last, saved), want))
    d = ssm.state_scan_bwd(u, dt, a_log, b, c, dy, saved, skip)
    want = ssm.state_scan_bwd(*few, some(dy), want[2], skip)
    assert all(torch.equal(some(getattr(d, k)), getattr(want, k)) for k in ("du", "ddt", "db", "dc"))
    del d, saved
    moved = some(last)
    one = ssm.state_scan_step(u[:, 0], dt[:, 0], a_log, b[:, 0], c[:, 0], last, skip)
    want = ssm.state_scan_step(few[0][:, 0], few[1][:, 0], a_log, few[3][:, 0], few[4][:, 0], moved, skip)
    assert torch.equal(some(one), want) and torch.equal(some(last), moved)
    w = torch.randn(D, 4, device="cuda")
    y, last = ssm.short_conv_fwd(u, w, want_state=True)
    want = ssm.short_conv_fwd(few[0], w, want_state=True)
    assert torch.equal(some(y), want[0]) and torch.equal(some(last), want[1])
    assert torch.equal(some(ssm.short_conv_bwd(u, w, None, dy)[0]), ssm.short_conv_bwd(few[0], w, None, some(dy))[0])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N", [(1, 16), (21, 5), (300, 16)])
def test_scan_steps_masked_by_infinities(device, dtype, T, N):
    """A step of softplus(-infinity), of the type's lowest value or of -300 is 0:
    the token changes no state.  NaN stays NaN."""
    p, dy, state, _ = scan_inputs(2, T, 12, N, 1, dtype, device, 41)
    gone = torch.rand(2, T, 12, generator=gen(5)).to(device) < 0.4

    def masked(value):
        q = dict(p, dt=torch.where(gone, torch.full_like(p["dt"], value), p["dt"]))
        y, last, saved = run_scan(q, state=state, want_state=True, save=True)
        return [y, last, *run_scan_bwd(q, dy, saved)]

    want = masked(-300.0)
    assert all(bool(torch.isfinite(v).all()) for v in want)
    for value in (-float("inf"), torch.finfo(dtype).min):
        assert all(torch.equal(a, b) for a, b in zip(masked(value), want))
    if T == 1:
        one = lambda v: v[:, 0]  # noqa: E731
        moved = state.clone()
        y = ssm.state_scan_step(one(p["u"]), torch.full_like(one(p["dt"]), -float("inf")), p["a_log"], one(p["b"]),
                                one(p["c"]), moved, p["skip"], one(p["z"]), p["dt_bias"])
        assert torch.equal(moved, state) and bool(torch.isfinite(y).all())
    p["dt"][0, 0, 3] = float("nan")
    y = run_scan(p)[0]
    assert bool(torch.isnan(y[0, :, 3]).all()) and bool(torch.isfinite(y[1]).all())
