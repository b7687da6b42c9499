"""Softmax cross entropy of a vocabulary projection at the ends of its range:
masks between the ordinary logits and fp32's lowest value, rows whose word is
certain, numbers of rows that a launch's grid has to hold.

The limits are those of `exact` in test_linear_cross_entropy.py unless a test
derives its own.
"""

import pytest
import torch

import dlvk_b200 as dl
from dlvk_b200.ops import core as K
from test_linear_cross_entropy import exact, near, operands

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e20, -1e30, -1e37, -1.9e38])
def test_words_masked_by_a_low_bias(device, dtype, low):
    """A bias of -1e4 and below leaves a word a probability of 0 (exp of less than -9000), whatever
    the number: a whole tile of such words adds nothing and spoils nothing."""
    x, w, t, b = operands(300, 64, 520, dtype, device, bias=True)
    b[500:] = low
    b[100:300] = low
    t = torch.where(t % 500 < 300, t % 100, t % 500)
    loss, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t, b)
    keep = torch.ones(520, dtype=torch.bool, device=device)
    keep[500:] = keep[100:300] = False
    where = torch.cumsum(keep, 0) - 1
    want = exact(x, w[:, keep], where[t], b[keep])
    near(loss, want["loss"], "loss")
    near(dl.LinearCrossEntropyLoss().forward(x, w, t, b), want["loss"], "loss alone")
    near(dx, want["dx"], "dx")
    near(dw[:, keep], want["dw"], "dw")
    near(db[keep], want["db"], "db")
    assert not dw[:, ~keep].any() and not db[~keep].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,v", [(12, 1040), (300, 1040), (2500, 9001)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("high", [12.0, 120.0, 1000.0, 2.0 ** 20, 2.0 ** 100])
def test_rows_whose_word_is_certain(device, dtype, n, v, bias, high):
    """Word 7 has a logit of high (1 to 2), the others 0: a loss of log(1 + (v - 1) e^-z).

    The row's maximum is its word's logit, so the loss is log(s) with s = 1 + the others' sum: never
    below 0.  s is a sum of v terms: off by 2^-24 of at most 2 for each of them, and each term by
    2^-22 (|z| + 2) of itself, as in `exact`.  Where e^-z is below fp32's smallest number, s is 1,
    the loss 0 and dz = 1 / s - 1 = 0."""
    g = torch.Generator().manual_seed(n)
    x, w = torch.zeros(n, 64, dtype=dtype, device=device), torch.zeros(64, v, dtype=dtype, device=device)
    x[:, 0] = (1 + torch.rand(n, generator=g)).to(dtype).to(device)
    w[0, 7] = high
    t = torch.full((n,), 7, dtype=torch.int32, device=device)
    b = torch.zeros(v, device=device) if bias else None
    rows = dl.LinearCrossEntropyLoss("none").forward(x, w, t, b)
    z = x[:, 0].double() * float(w[0, 7])
    others = (v - 1) * torch.exp(-z)
    want = torch.log1p(others)
    # z itself is a product rounded to fp32
    lim = (v + 2) * 2.0 ** -23 + others * (2.0 ** -22 * (z + 2) + 2.0 ** -24 * z)
    assert bool((rows >= 0).all()), float(rows.min())
    assert bool(((rows.double() - want).abs() <= lim).all()), float((rows.double() - want).abs().max())
    loss, dx, dw, db = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t, b)
    assert float(loss) >= 0 and abs(float(loss) - float(want.mean())) <= float(lim.mean()) + 2.0 ** -24 * float(loss)
    if high > 104:
        assert float(loss) == 0.0 and not dx.any() and not dw.any() and (db is None or not db.any())


@pytest.mark.parametrize("room", [1 << 26, 1 << 27, 1 << 30])  # fp32 logits, exponentials, statistics alone
@pytest.mark.parametrize("classes", [1, 2, 5, 15, 63, 64, 65, 127, 1000, 4096, 50257, 65537, 151936, 2 ** 30 - 1])
def test_blocks_of_rows_fit_every_launch(classes, room):
    """Passes over a block have a grid of rows / 32 or rows / 64 in its second dimension: at most 65535."""
    f = dl._ext.C().linear_ce_block_rows
    for rows in (1, 31, 255, 2048, 2049, 2 ** 20 - 1, 2 ** 20 + 1, 2 ** 21, 2 ** 22, 4470000, 2 ** 26, 2 ** 31 - 257):
        n = f(rows, classes, room)
        assert 1 <= n <= rows and (n == rows or n % 256 == 0)
        assert -(-n // 32) <= 65535
        line = -(-classes // 64) * 64
        # equal blocks of whole tiles: at most a tile's rows above the room
        assert n * line <= max(2048 * line, room) + 256 * line


def in_parts(x, w, t, b, parts):
    """What `check` compares, with the 64-bit values made of a part of the rows at a time."""
    loss, dx, dw, db = dl.LinearCrossEntropyLoss("sum").value_and_grad(x, w, t, b)
    rows = dl.LinearCrossEntropyLoss("none").forward(x, w, t, b)
    n, total = x.shape[0], {}
    for i in range(parts):
        s = slice(i * n // parts, (i + 1) * n // parts)
        want = exact(x[s], w, t[s], b, mean=False)
        near(rows[s], want["rows"], "rows")
        near(dx[s], want["dx"], "dx")
        for k in ("loss", "dw", "db"):
            value, lim = total.get(k, (0.0, 0.0))
            # the whole sum has `parts` times the additions that a part's limit counts
            total[k] = value + want[k][0], lim + parts * want[k][1]
    near(loss, total["loss"], "loss")
    near(dw, total["dw"], "dw")
    if b is not None:
        near(db, total["db"], "db")


@pytest.mark.gpu
def test_two_million_rows_of_64_words():
    in_parts(*operands(2 ** 21, 16, 64, torch.bfloat16, "cuda"), 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_millions_of_rows_of_a_few_words(dtype):
    """Logits by the SIMT product: 64 rows to a block."""
    in_parts(*operands(4300000, 8, 5, dtype, "cuda", bias=True), 10)


@pytest.mark.gpu
def test_millions_of_words_of_a_few_numbers():
    """dW of a tied table by the SIMT product: a row of it per word, 64 to a block."""
    n, e, v = 20, 4, 4300000
    x, w, t, _ = operands(n, e, v, torch.float32, "cuda", tied=True)
    t[0] = v - 1
    want = exact(x, w, t, None)
    loss, dx, dw, _ = dl.LinearCrossEntropyLoss().value_and_grad(x, w, t)
    near(loss, want["loss"], "loss")
    near(dx, want["dx"], "dx")
    near(dw, want["dw"], "dw")


@pytest.mark.gpu
def test_refusals_of_gradients_that_repeat_or_lie_on_operands():
    x, w, t, b = operands(40, 1, 70, torch.float32, "cuda", bias=True)
    with pytest.raises(RuntimeError, match="repeats"):  # one row, one element for all words
        K.linear_ce(x, w, t, b, dw_out=torch.zeros(1, 1, device="cuda").expand(1, 70))
    x, w, t, b = operands(40, 16, 1, torch.float32, "cuda", bias=True)
    with pytest.raises(RuntimeError, match="repeats"):
        K.linear_ce(x, w, t, b, dw_out=torch.zeros(1, 1, device="cuda").expand(16, 1))
    out = torch.zeros(16, 3, device="cuda")[:, :1]  # rows apart: one column of a wider matrix
    K.linear_ce(x, w, t, b, dw_out=out)
    x, w, t, b = operands(40, 16, 70, torch.float32, "cuda", bias=True)
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(x, w, t, b, db_out=b)
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(x, w, t, b, db_out=w[0])
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(x, w, t, b, db_out=x.reshape(-1)[:70])
    both = torch.zeros(16 * 70 + 70, device="cuda")
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(x, w, t, b, dw_out=both[:1120].view(16, 70), db_out=both[1100:1170])
    with pytest.raises(RuntimeError, match="memory"):
        K.linear_ce(x, w, t, both[1000:1070], dw_out=both[:1120].view(16, 70))
    K.linear_ce(x, w, t, b, dw_out=both[:1120].view(16, 70), db_out=both[1120:])
    want = exact(x, w, t, b)
    near(both[:1120].view(16, 70), want["dw"], "dw")
    near(both[1120:], want["db"], "db")
