"""Softmax cross entropy of a vocabulary projection without its logits.

Every limit below is a bound on the arithmetic, taken elementwise in 64 bits
from the same inputs:

* a logit is an fp32 sum of `width` products of exact operands (and the bias):
  off by dz <= (width + 2) * 2^-23 * sum |x w| (each addition may truncate); fp32 operands on the
  tensor cores are split in two parts of 11 bits, which leaves 2^-20 of each
  product out;
* a probability is exp of (z - lse): off by the errors of both, 2^-22 (|z| +
  |lse| + 2) for the roundings of the exponent, the table-free exp2 and the
  sum's, relative;
* without a bias, bf16 operands keep exp(z - local maximum) as fp16 times 2^15: 2^-11 of it,
  and 2^-40 of the largest where it is that small;
* dz = (p - onehot) g is rounded to bf16 (2^-8) where the operands are bf16;
* dx, dW are fp32 sums of those (2^-23 per addition of their magnitude) and one
  rounding to their type; db is an fp32 sum of unrounded dz.
"""
import math

import pytest
import torch

import dlvk_b200 as dl
from dlvk_b200.models.sequential import Sequential
from dlvk_b200.ops import core as K

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
U = 2.0 ** -23


def operands(n, e, v, dtype, device, tied=False, bias=False, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(v, e, generator=g) * (spread / math.sqrt(e))
    x = torch.randn(n, e, generator=g)
    t = torch.randint(0, v, (n,), generator=g)
    x += 2.0 * (torch.rand(n, 1, generator=g) < 0.4) * w[t]
    b = torch.randn(v, generator=g).to(device) if bias else None
    w = w.to(dtype).to(device)
    return x.to(dtype).to(device), (w.t() if tied else w.t().contiguous()), t.to(device), b


def exact(x, w, t, b, mean=True, ignore=None, scale=1.0):
    """Values and limits in 64 bits: {"loss", "rows", "dx", "dw", "db"} -> (value, limit)."""
    bf = x.dtype == torch.bfloat16
    N, V = x.shape[0], w.shape[1]
    counted = (t >= 0) & (t < V)
    if ignore is not None:
        counted &= t != ignore
    X, W, lab = x.double()[counted], w.double(), t.long()[counted]
    bb = b.double() if b is not None else torch.zeros(V, dtype=torch.float64, device=x.device)
    z = X @ W + bb
    mag = X.abs() @ W.abs() + torch.where(bb.isfinite(), bb.abs(), torch.zeros_like(bb))
    dz_ = ((X.shape[1] + 2) * U + (0 if bf else 2.0 ** -20)) * mag
    lse = torch.logsumexp(z, -1)
    top = dz_.amax(-1) if V else lse
    i = torch.arange(lab.numel(), device=x.device)
    rows = torch.zeros(N, dtype=torch.float64, device=x.device)
    rlim = torch.zeros_like(rows)
    rows[counted] = lse - z[i, lab]
    rlim[counted] = top + dz_[i, lab] + 2.0 ** -22 * (lse.abs() + z[i, lab].abs() + 2)
    m = lab.numel()
    share = (1.0 / max(m, 1)) if mean else 1.0
    g = share * scale
    p = torch.exp(z - lse[:, None])
    zf = torch.where(z.isfinite(), z.abs(), torch.zeros_like(z))
    perr = p * (dz_ + top[:, None] + 2.0 ** -22 * (zf + lse.abs()[:, None] + 2))
    d = p.clone()
    d[i, lab] -= 1.0
    if bf and b is None and m:
        perr = perr + 2.0 ** -11 * p + 2.0 ** -40 * p.amax(-1, keepdim=True)
    # 2^-22: the subtraction and the product by g
    derr = (perr + 2.0 ** -22 * (p + d.abs())) * g
    d *= g
    dq = derr + (HALF[x.dtype] * (d.abs() + derr) if bf else 0)
    tf = 0 if bf else 2.0 ** -20
    dx, xlim = torch.zeros_like(X), None
    dx = d @ W.t()
    xlim = dq @ W.abs().t() + ((V + 2) * U + tf) * (d.abs() @ W.abs().t())
    dw = X.t() @ d
    wlim = X.abs().t() @ dq + ((m + 2) * U + tf) * (X.abs().t() @ d.abs())
    full = torch.zeros(N, X.shape[1], dtype=torch.float64, device=x.device)
    flim = torch.zeros_like(full)
    full[counted], flim[counted] = dx, xlim
    tiny = 1e-37
    # the sum of the losses is kept in 64 bits and rounded once
    return {"loss": (rows.sum() * share, rlim.sum() * share + 2.0 ** -24 * rows.abs().sum() * share + tiny),
            "rows": (rows, rlim + 2.0 ** -24 * rows.abs() + tiny),
            "dx": (full, flim + HALF[x.dtype] * (full.abs() + flim) + tiny),
            "dw": (dw, wlim + HALF[w.dtype] * (dw.abs() + wlim) + tiny),
            "db": (d.sum(0), derr.sum(0) + (m + 2) * U * d.abs().sum(0) + tiny)}


def near(got, want, what):
    ref, lim = want
    over = (got.double() - ref).abs() - lim
    assert bool((over <= 0).all()), (what, float(over.max()), float(ref.abs().max()))


def check(x, w, t, b, mean=True, ignore=None, want_layout=True):
    loss_fn = dl.LinearCrossEntropyLoss("mean" if mean else "sum", ignore)
    want = exact(x, w, t, b, mean, ignore)
    loss, dx, dw, db = loss_fn.value_and_grad(x, w, t, b)
    assert loss.dtype == torch.float32 and dx.dtype == x.dtype and dw.dtype == w.dtype
    assert dx.shape == x.shape and dw.shape == w.shape
    near(loss, want["loss"], "loss")
    near(dx, want["dx"], "dx")
    near(dw, want["dw"], "dw")
    if b is not None:
        assert db.dtype == torch.float32
        near(db, want["db"], "db")
    else:
        assert db is None
    near(loss_fn.forward(x, w, t, b), want["loss"], "loss alone")
    near(dl.LinearCrossEntropyLoss("none", ignore).forward(x, w, t, b), want["rows"], "rows")
    return loss, dx, dw, db


SHAPES = [(1, 8, 64), (2, 64, 65), (5, 16, 100), (33, 64, 129), (128, 24, 64), (129, 200, 255), (255, 40, 300),
          (256, 64, 1000), (257, 128, 513), (300, 72, 4099), (512, 256, 1024)]
ODD = [(1, 1, 1), (3, 2, 1), (4, 1, 2), (7, 5, 10), (40, 33, 70), (64, 31, 333), (260, 65, 999), (300, 129, 1003)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shape", SHAPES + ODD)
def test_values(device, dtype, tied, bias, shape):
    x, w, t, b = operands(*shape, dtype, device, tied, bias, seed=sum(shape))
    if shape[0] > 2:
        t[1] = -1
        t[2] = shape[2]  # outside: does not count either
    check(x, w, t.to(torch.int32) if tied else t, b, mean=bias or shape[0] < 100)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_several_blocks(dtype, tied, bias):
    # 33000 / 20000 rows of 5003 classes are two blocks
    x, w, t, b = operands(33000 if dtype == torch.bfloat16 else 20000, 16, 5003, dtype, "cuda", tied, bias)
    t[::7] = -1
    check(x, w, t, b)
    W = torch.ones_like(w, dtype=torch.float32)
    K.linear_ce(x, w, t, b, dw_out=W, dw_accumulate=True)
    ref, lim = exact(x, w, t, b)["dw"]
    near(W, (1.0 + ref, lim + 2.0 ** -22 * (1 + ref.abs())), "accumulated")


@pytest.mark.gpu
def test_loss_alone_in_several_blocks():
    # 2^30 / 60000 rows: three blocks, and a last one of 40 rows
    n = 2 * 8960 + 40
    x, w, t, _ = operands(n, 8, 120000, torch.bfloat16, "cuda", True)
    rows = dl.LinearCrossEntropyLoss("none").forward(x, w, t)
    for part in (slice(0, 300), slice(8900, 9000), slice(n - 50, n)):
        near(rows[part], exact(x[part], w, t[part], None, mean=False)["rows"], "rows")
    mean = dl.LinearCrossEntropyLoss().forward(x, w, t)
    assert abs(float(mean) - float(rows.double().mean())) <= 2.0 ** -23 * float(mean)


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,e,v", [(1, 520, 9001), (3, 1031, 2000), (4, 64, 70001), (8, 96, 11361), (16, 515, 5000),
                                   (17, 40, 3001), (31, 700, 12000), (32, 1500, 800), (33, 128, 4000),
                                   (2, 512, 60000), (20, 33, 60001)])
def test_few_rows_of_fp32(tied, n, e, v):
    x, w, t, b = operands(n, e, v, torch.float32, "cuda", tied, n % 2 == 0)
    check(x, w, t, b)
    W = torch.ones_like(w)
    K.linear_ce(x, w, t, b, dw_out=W, dw_accumulate=True)
    ref, lim = exact(x, w, t, b)["dw"]
    near(W, (1.0 + ref, lim + 2.0 ** -22 * (1 + ref.abs())), "accumulated")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [100, 700])
def test_long_rows_and_wide(rows):
    x, w, t, b = operands(rows, 1032, 20001, torch.bfloat16, "cuda", True, False)
    check(x, w, t, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_do_not_count(device, dtype):
    """Padding rows hold whatever they hold: NaN and infinities there reach nothing."""
    x, w, t, b = operands(300, 64, 520, dtype, device, bias=True)
    out = torch.zeros(300, dtype=torch.bool, device=device)
    out[[0, 5, 64, 127, 128, 299]] = True
    t = torch.where(out, torch.full_like(t, -100), t)
    clean = x.clone()
    clean[out] = 0
    ref = check(clean, w, t, b)
    dirty = x.clone()
    dirty[out] = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=device).repeat(16).to(dtype)
    got = dl.LinearCrossEntropyLoss().value_and_grad(dirty, w, t, b)
    assert all(torch.equal(a, c) for a, c in zip(got, ref)) and not got[1][out].any()
    rows = dl.LinearCrossEntropyLoss("none").forward(dirty, w, t, b)
    assert not rows[out].any() and bool(rows.isfinite().all())
    # a word that does not count
    word = int(t[~out][0])
    check(clean, w, t, b, ignore=word)
    # none counts
    loss, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(dirty, w, torch.full_like(t, -1), b)
    assert float(loss) == 0.0 and not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min])
def test_masked_words(device, dtype, low):
    """Words that a bias rules out (padding of the vocabulary) have probability and gradients 0."""
    x, w, t, b = operands(300, 64, 520, dtype, device, bias=True)
    t = t % 500
    b[500:] = low
    b[100:300] = low
    t = torch.where((t >= 100) & (t < 300), t % 100, t)
    loss, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t, b)
    keep = torch.ones(520, dtype=torch.bool, device=device)
    keep[500:] = keep[100:300] = False
    where = torch.cumsum(keep, 0) - 1
    want = exact(x, w[:, keep], where[t], b[keep])
    near(loss, want["loss"], "loss")
    near(dx, want["dx"], "dx")
    near(dw[:, keep], want["dw"], "dw")
    near(db[keep], want["db"], "db")
    assert not dw[:, ~keep].any() and not db[~keep].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_word_masked_by_the_lowest_value(device, dtype):
    """z = -3.4e38 for every word (what x W adds is lost there): equal probabilities."""
    x, w, t, b = operands(300, 64, 520, dtype, device, bias=True)
    b.fill_(torch.finfo(torch.float32).min)
    loss, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t, b)
    even = exact(x, torch.zeros_like(w), t, torch.zeros_like(b))
    assert abs(float(loss) - math.log(520)) <= 2.0 ** -21 * math.log(520)
    near(db, even["db"], "db")
    near(dw, even["dw"], "dw")


@pytest.mark.parametrize("device", DEVICES)
def test_far_logits_and_nan(device):
    x, w, t, _ = operands(200, 64, 300, torch.bfloat16, device, spread=60.0)
    check(x, w, t, None)  # logits of hundreds: probabilities of 0 and 1
    x[7, 3] = math.nan
    loss, dx, dw, _ = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t)
    assert math.isnan(float(loss)) and bool(dx[7].isnan().all()) and bool(dx[8].isfinite().all())
    rows = dl.LinearCrossEntropyLoss("none").forward(x, w, t)
    assert bool(rows[7].isnan()) and int(rows.isnan().sum()) == 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(device, dtype):
    n, e, v = 270, 48, 200
    x, w, t, _ = operands(n, e, v, dtype, device)
    wide = torch.zeros(n, 3 * e, dtype=dtype, device=device)
    wide[:, 5:5 + e] = x
    tall = torch.zeros(e, 2 * v + 1, dtype=dtype, device=device)
    tall[:, 1:1 + v] = w
    spaced = torch.zeros(e, 2 * v, dtype=dtype, device=device)
    spaced[:, ::2] = w
    ref = check(x, w, t, None)
    for xv, wv in ((wide[:, 5:5 + e], tall[:, 1:1 + v]), (x.t().contiguous().t(), spaced[:, ::2]),
                   (x, torch.cat([w.t(), w.t()])[:v].t())):
        check(xv, wv, t, None)
    check(x[:1].expand(n, e), w, t, None)  # one row for all
    loss, dx, dw, _ = dl.LinearCrossEntropyLoss().value_and_grad(x.reshape(27, 10, e), w, t.reshape(27, 10))
    assert dx.shape == (27, 10, e) and torch.equal(dx.reshape(n, e), ref[1]) and torch.equal(dw, ref[2])
    spread = torch.stack([t, t], 1)[:, 0]
    assert torch.equal(dl.LinearCrossEntropyLoss().value_and_grad(x, w, spread)[1], ref[1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,v", [(4, 16, 40), (24, 64, 3001), (300, 64, 1024)])
@pytest.mark.parametrize("bias", [False, True])
def test_logits_near_the_largest_value(device, dtype, n, e, v, bias):
    """One word's logit is 1.875 * 2^127 = 3.19e38, whose product with log2 e
    is above fp32: losses 0 and 3.19e38, probabilities 1 and 0."""
    x, w = torch.zeros(n, e, dtype=dtype, device=device), torch.zeros(e, v, dtype=dtype, device=device)
    x[:, 0], w[0, 5] = 1.5 * 2.0 ** 64, 1.25 * 2.0 ** 63
    t = torch.full((n,), 5, dtype=torch.int32, device=device)
    t[1::2] = 1
    b = torch.zeros(v, device=device) if bias else None
    rows = dl.LinearCrossEntropyLoss("none").forward(x, w, t, b)
    assert bool((rows[0::2] == 0).all()) and bool((rows[1::2] == 1.875 * 2.0 ** 127).all())
    _, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t, b)
    odd = n // 2
    want_x, want_w = torch.zeros(n, e, dtype=torch.float64), torch.zeros(e, v, dtype=torch.float64)
    want_x[1::2, 0] = 1.25 * 2.0 ** 63 / n
    want_w[0, 5], want_w[0, 1] = odd / n * 1.5 * 2.0 ** 64, -odd / n * 1.5 * 2.0 ** 64
    # 1 / n and the products: a handful of fp32 roundings, and for dW one for each
    # of the `odd` equal terms of a sum; one to the type of the output
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    for got, want, terms in ((dx, want_x, 1), (dw, want_w, odd)):
        assert bool(((got.double().cpu() - want).abs() <= (half + (terms + 8) * 2.0 ** -24) * want.abs()).all())
    if bias:
        want_b = torch.zeros(v, dtype=torch.float64)
        want_b[5], want_b[1] = odd / n, -odd / n
        assert bool(((db.double().cpu() - want_b).abs() <= (odd + 8) * 2.0 ** -24 * want_b.abs()).all())


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows(device):
    x, w, t, b = operands(3, 16, 70, torch.bfloat16, device, bias=True)
    loss, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(x[:0], w, t[:0], b)
    assert float(loss) == 0.0 and dx.shape == (0, 16) and not dw.any() and not db.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_given_scaled_and_counted(device, dtype):
    x, w, t, b = operands(300, 64, 521, dtype, device, bias=True)
    want = exact(x, w, t, b, scale=8.0)
    W = torch.ones(64, 521, device=device)
    B = torch.ones(521, device=device)
    hits = torch.full((1,), 5, dtype=torch.int64, device=device)
    eight = torch.tensor([8.0], device=device)
    K.linear_ce(x, w, t, b, grad_scale=eight, dw_out=W, dw_accumulate=True, db_out=B, db_accumulate=True, correct=hits)
    # an fp32 output is not rounded to bf16; the sum with what was there is one more rounding
    for got, (ref, lim) in ((W, want["dw"]), (B, want["db"])):
        near(got, (1.0 + ref, lim + 2.0 ** -22 * (1 + ref.abs())), "accumulated")
    K.linear_ce(x, w, t, b, grad_scale=eight, dw_out=W, db_out=B)
    near(W, want["dw"], "overwritten")
    near(B, want["db"], "overwritten")
    z = x.double() @ w.double() + b.double()
    assert int(hits) == 5 + int((z.argmax(1) == t).sum())


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    """(L(x + h d) - L(x - h d)) / 2h against <dx, d>: the third derivative of log sum exp
    along d is a third cumulant, at most R^3 for logits that move within R; the losses'
    roundings are divided by 2h."""
    x, w, t, b = operands(20, 16, 80, torch.float32, device, bias=True)
    fn = dl.LinearCrossEntropyLoss("sum")
    _, dx, dw, db = fn.value_and_grad(x, w, t, b)
    g = torch.Generator().manual_seed(9)
    h = 2.0 ** -6
    for which in range(3):
        d = [torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)]
        d[which] = (torch.randn(d[which].shape, generator=g).to(device) / 4)
        up = [p + h * q for p, q in zip((x, w, b), d)]
        dn = [p - h * q for p, q in zip((x, w, b), d)]
        diff = (float(fn.forward(up[0], up[1], t, up[2]).double()) - float(fn.forward(dn[0], dn[1], t, dn[2]).double())) / (2 * h)
        move = x.double() @ d[1].double() + d[0].double() @ w.double() + d[2].double()
        R = float((move.amax(1) - move.amin(1)).max())
        want = sum(float((a.double() * q.double()).sum()) for a, q in zip((dx, dw, db), d))
        lim = float(exact(up[0], up[1], t, up[2], mean=False)["loss"][1] + exact(dn[0], dn[1], t, dn[2], mean=False)["loss"][1])
        lims = exact(x, w, t, b, mean=False)
        slack = sum(float((lims[k][1] * q.abs()).sum()) for k, q in zip(("dx", "dw", "db"), d))
        # x + h d is rounded to fp32 too: 2^-24 of it, times the gradient
        slack += sum(float((a.abs() * p.abs()).sum()) * 2.0 ** -23 / h for a, p in zip((dx, dw, db), (x, w, b)))
        assert abs(diff - want) <= h * h / 6 * 20 * R ** 3 + lim / (2 * h) + slack


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, t, b = operands(6, 16, 70, torch.bfloat16, device, bias=True)
    fn = dl.LinearCrossEntropyLoss()
    E = (ValueError, RuntimeError)
    for args in ((x, w[:8], t), (x, w.float(), t), (x.half(), w.half(), t), (x, w, t[:5]), (x, w, t.float()),
                 (x, w, t, b[:69]), (x, w[:, :0], t)):
        with pytest.raises(E):
            fn.value_and_grad(*args)
    with pytest.raises(ValueError):
        dl.LinearCrossEntropyLoss("average")
    with pytest.raises(ValueError):
        dl.LinearCrossEntropyLoss("none").value_and_grad(x, w, t)
    m = Sequential(device if device == "cpu" else "cuda:0", "fp32", seed=0)
    m.add_dense(8, 4).add_relu()
    with pytest.raises(ValueError, match="Dense"):
        m.train_step(torch.randn(2, 8), torch.zeros(2, dtype=torch.int32), fn, dl.SGD(0.1))


def test_evaluation_needs_one_loss():
    m = Sequential("cpu", "fp32", seed=0)
    m.add_dense(8, 70)
    x, y = torch.randn(2, 8), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="reduction"):
        m.head_loss(x, y, dl.LinearCrossEntropyLoss("none"))
    loss, hits, rows = m.head_loss(x, y, dl.LinearCrossEntropyLoss("sum"))
    assert rows == 2 and 0 <= hits <= 2 and float(loss) > 0


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, w, t, b = operands(6, 16, 70, torch.bfloat16, "cuda", bias=True)
    with pytest.raises(RuntimeError, match="target"):
        K.linear_ce(x, w, t.cpu())
    with pytest.raises(RuntimeError, match="weight"):
        K.linear_ce(x, w.cpu(), t)
    with pytest.raises(RuntimeError, match="weight gradient"):
        K.linear_ce(x, w, t, dw_out=torch.zeros(16, 71, device="cuda"))
    with pytest.raises(RuntimeError, match="weight gradient"):
        K.linear_ce(x, w, t, dw_out=torch.zeros_like(w), dw_accumulate=True)
    with pytest.raises(RuntimeError, match="bias gradient"):
        K.linear_ce(x, w, t, db_out=torch.zeros(70, device="cuda"))
    with pytest.raises(RuntimeError, match="grad_scale"):
        K.linear_ce(x, w, t, grad_scale=torch.ones(2, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K_", [(160, 512, 256), (33, 256, 64), (1056, 1024, 512), (8224, 1024, 256)])
def test_column_sums_of_a_product_with_part_tiles(M, N, K_):
    """The products' column sums where the last tile has whole 32-row chunks
    past M: those write nowhere, and the sums are those of the rows there are."""
    C = K.N()
    g = torch.Generator(device="cuda").manual_seed(3)
    a = torch.randn(M, K_, device="cuda", generator=g).bfloat16()
    b = (torch.randn(K_, N, device="cuda", generator=g) * 0.1).bfloat16()
    cs = torch.full((N,), 7.0, device="cuda")
    out = C.gemm(a, b, out_dtype=torch.float32, colsum_out=cs)
    want = out.double().sum(0)
    # fp32 sums of M terms in whatever order: at most M 2^-24 of the sum of magnitudes
    lim = M * 2.0 ** -24 * out.double().abs().sum(0)
    assert bool(((cs.double() - want).abs() <= lim).all())
    assert int(C.read_device_error(True)) == 0


@pytest.mark.gpu
def test_refusals_of_a_weight_gradient_on_other_memory():
    x, w, t, _ = operands(6, 16, 70, torch.float32, "cuda")
    wide = torch.zeros(16, 70, device="cuda")
    for bad in (wide[:1].expand(16, 70), wide.as_strided((16, 70), (69, 1)), wide.as_strided((16, 70), (1, 15))):
        with pytest.raises(RuntimeError, match="repeats"):
            K.linear_ce(x, w, t, dw_out=bad)
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(x, w, t, dw_out=w)
    both = torch.zeros(6 * 16 + 16 * 70, device="cuda")
    h = both[:96].view(6, 16)
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(h, w, t, dw_out=both[80:80 + 1120].view(16, 70))


def _token_model(device, dtype, vocab=300, hidden_relu=False, bias=False):
    m = Sequential(device if device == "cpu" else "cuda:0", dtype, seed=3)
    m.add_embedding(vocab, 64, init_std=0.5, embed_scale=2.0, padding_idx=0)
    m.add_layernorm(64)
    if hidden_relu:
        m.add_dense(64, 128).add_relu()
    m.add_dense(128 if hidden_relu else 64, vocab, use_bias=bias, init_std=0.1)
    m.add_softmax()
    return m.build()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("relu,bias", [(False, False), (True, True)])
def test_model_gradients_are_those_of_the_unfused_loss(device, relu, bias):
    """fp32 model: the same step through CrossEntropyLoss.  Both sums are fp32 sums of the
    same terms (through split products on the GPU): 1e-4 of each gradient's largest value is
    far above (300 + 300) * 2^-20 = 6e-4 of a typical one's 1/6."""
    a, b = _token_model(device, "fp32", hidden_relu=relu, bias=bias), _token_model(device, "fp32", hidden_relu=relu, bias=bias)
    x = torch.randint(0, 300, (4, 25), dtype=torch.int32)
    y = torch.randint(0, 300, (4, 25), dtype=torch.int32)
    la = a.train_step(x, y, dl.CrossEntropyLoss(), dl.SGD(0.0))
    lb = b.train_step(x, y, dl.LinearCrossEntropyLoss(), dl.SGD(0.0))
    assert abs(float(la) - float(lb)) <= 1e-5 * float(la)
    for p, q in zip(a.parameters(), b.parameters()):
        assert float((p.grad - q.grad).abs().max()) <= 1e-4 * float(p.grad.abs().max()), p.name
    with pytest.raises(RuntimeError):
        b.backward(torch.zeros(1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_the_operators_in_one_captured_step(dtype):
    """Embedding, head loss, clipping and update as a training step uses them: a captured
    TrainStep gives the eager step's parameters bit for bit, at every step."""
    steps = []
    for graph in (False, True):
        m = _token_model("cuda", dtype)
        opt = dl.Adam(1e-3)
        opt.set_gradient_clipping(max_norm=0.05)
        steps.append(dl.TrainStep(m, dl.LinearCrossEntropyLoss(), opt, graph=graph, metrics=True))
    g = torch.Generator().manual_seed(1)
    for _ in range(6):
        x = torch.randint(0, 300, (8, 40), generator=g, dtype=torch.int32)
        y = torch.randint(-1, 300, (8, 40), generator=g, dtype=torch.int32)
        losses = [s(x, y).item() for s in steps]
        assert losses[0] == losses[1]
        norms = [float(dl.GradientClipping.global_norm([p.grad for p in s.model.parameters()])) for s in steps]
        assert norms[0] == norms[1] and norms[0] > 0.05
        for p, q in zip(*(s.model.parameters() for s in steps)):
            assert torch.equal(p.grad, q.grad) and torch.equal(p.master, q.master)
    assert steps[1].replays > 0 and steps[0].epoch_metrics() == steps[1].epoch_metrics()
    for s in steps:
        s.close()


@pytest.mark.gpu
def test_an_eager_graph_of_the_model_may_live_during_capture():
    m = _token_model("cuda", "bf16")
    x = torch.randint(0, 300, (8, 40), dtype=torch.int32)
    kept = m.forward(x)  # its autograd graph stays alive
    step = dl.TrainStep(m, dl.LinearCrossEntropyLoss(), dl.SGD(1e-2))
    for _ in range(4):
        loss = step(x, x)
    assert math.isfinite(loss.item()) and step.replays > 0 and kept.requires_grad
    step.close()


@pytest.mark.parametrize("device", DEVICES)
def test_loss_scale_and_trainers(device):
    """A scaled step updates as an unscaled one (the scale is a power of 2), and fit /
    evaluate take the loss."""
    dev = device if device == "cpu" else "cuda:0"
    x = torch.randint(1, 300, (32, 10), dtype=torch.int32)
    models = []
    for scaled in (False, True):
        m = _token_model(device, "fp32")
        scaler = dl.GradientScaler(init_scale=1024.0, device=dev) if scaled else None
        step = dl.TrainStep(m, dl.LinearCrossEntropyLoss(), dl.SGD(0.1), scaler=scaler)
        for _ in range(3):
            step(x, x)
        models.append(m)
        step.close()
    for p, q in zip(*(m.parameters() for m in models)):
        assert float((p.master - q.master).abs().max()) <= 1e-5 * float(p.master.abs().max())
    tr = dl.ModelTrainer(models[0])
    tr.compile(dl.Adam(1e-2), dl.LinearCrossEntropyLoss())
    hist = tr.fit(x, x, epochs=2, batch_size=16, verbose=False, validation_split=0.25)
    m = tr.evaluate(x, x, 16)
    assert math.isfinite(hist[-1].loss) and 0.0 <= hist[-1].accuracy <= 1.0 and 0.0 <= m.accuracy <= 1.0
    assert math.isfinite(m.loss)


@pytest.mark.gpu
def test_same_bits_every_time_and_on_another_stream():
    x, w, t, b = operands(5000, 256, 9001, torch.bfloat16, "cuda", True, True)
    fn = dl.LinearCrossEntropyLoss()
    first = fn.value_and_grad(x, w, t, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            again = fn.value_and_grad(x, w, t, b)
        other = fn.value_and_grad(x, w, t, b)  # at the same time
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        assert all(torch.equal(p, q) for p, q in zip(first, other))
    W = [torch.zeros(9001, 256, device="cuda") for _ in range(2)]
    for o in W:
        K.linear_ce(x, w, t, b, dw_out=o.t())
    assert torch.equal(*W)
    assert dl._ext.C().read_device_error(True) == 0
