"""The fp32 products of the vocabulary cross entropy on the tensor cores: operands
in three bf16 parts, x = x0 + x1 + x2, of whose nine products the six that reach
above 2^-24 of the whole are made.

Sums of one term: what a product is then off by is its arithmetic alone, with no
sum's roundings beside it:

* the three products left out: at most 2 * 2^-9 * 2^-17 + 2^-34 < 2^-24 of the
  whole (a part is at most 2^-8 of the one before it, and what rounding leaves
  of that half);
* five small products in one fp32 accumulator, at most 2^-8 + 2^-8 + ... < 2^-6 of
  the whole, each addition truncated: 5 * 2^-23 * 2^-6;
* their sum with x0 w0 (exact) and the scaling, by 1: 2 * 2^-24.

Below 2^-22 in all.  A product that is lost shows: for each of the six the test
first makes the sum without it on the CPU and sees that it is off by four limits
somewhere.

Sums of many terms: one large term first, then terms of 2^-29 of it.  An
accumulator that holds the large one loses the others whole (they are below half
of its last place); every other accumulator sums them exactly.  So the loss counts
the terms that share the large one's accumulator.
"""
import pytest
import torch

import dlvk_b200 as dl

pytestmark = pytest.mark.gpu
LIMIT = 2.0 ** -22
SIZES = [(1024, 64, 261), (300, 600, 1300), (2300, 128, 997), (40, 700, 1003), (700, 1400, 331)]


def parts(t):
    a = t.float().bfloat16().float()
    b = (t.float() - a).bfloat16().float()
    return [p.double() for p in (a, b, (t.float() - a - b).bfloat16().float())]


def fine(n, seed):
    """Numbers in [1, 2) with 24 bits, of either sign."""
    g = torch.Generator().manual_seed(seed)
    v = 1 + torch.randint(0, 2 ** 23, (n,), generator=g).double() * 2.0 ** -23
    return (v * (1 - 2 * torch.randint(0, 2, (n,), generator=g))).float().cuda()


def near(got, x, w, sees=True):
    """got = x w to LIMIT; first that the limit sees each of the six products."""
    want = x.double() * w.double()
    p, q = parts(x), parts(w)
    for i in range(3):
        for j in range(3 - i):
            assert not sees or bool(((p[i] * q[j]).abs() > 4 * LIMIT * want.abs()).any()), (i, j)
    over = (got.double() - want).abs() - LIMIT * want.abs()
    assert bool((over <= 0).all()), float((over / want.abs()).max())


def three_parts(v):
    """Whether 1 / v has three parts that the limit sees (1 / 261's third is below 2^-21 of it, 1 / 331's second 2^-15)."""
    return v not in (261, 331)


def laid_out(w, tied):
    return w.t().contiguous().t() if tied else w


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,e,v", SIZES)
def test_every_product_of_the_logits(n, e, v, tied):
    """Word 7's logit is a single product of 64 and more, the others 0, the label another
    word: a loss of z + log(1 + (v - 1) e^-z), the last of which is below 2^-80 z."""
    x, w = torch.zeros(n, e, device="cuda"), torch.zeros(e, v, device="cuda")
    col = torch.arange(n, device="cuda") % e
    a, b = fine(n, 1).abs(), fine(e, 2).abs()
    x[torch.arange(n, device="cuda"), col] = a
    w[:, 7] = b * 64
    t = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    near(dl.LinearCrossEntropyLoss("none").forward(x, laid_out(w, tied), t), a, b[col] * 64)
    # with gradients the logits go another way: the mean of n equal losses, row after row the same
    for k in range(0, n, max(1, n // 4)):
        same = x[k:k + 1].expand(n, e).contiguous()
        loss = dl.LinearCrossEntropyLoss().value_and_grad(same, laid_out(w, tied), t)[0]
        want = float(a[k].double() * b[col[k]].double() * 64)
        assert abs(float(loss) - want) <= (LIMIT + 2.0 ** -24) * want


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,e,v", SIZES)
def test_every_product_of_dx(n, e, v, tied):
    """x = 0: every word's probability is 1 / v, rounded once (1 / s; s counts exactly).  dx of
    column c is that times the one word of it that has a number."""
    x = torch.zeros(n, e, device="cuda")
    w = torch.zeros(e, v, device="cuda")
    word = 4 + torch.arange(e, device="cuda") % (v - 4)
    b = fine(e, 3)
    w[torch.arange(e, device="cuda"), word] = b
    t = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    dx = dl.LinearCrossEntropyLoss("sum").value_and_grad(x, laid_out(w, tied), t)[1]
    p = torch.full((e,), 1.0 / v, device="cuda")
    near(dx[0], p, b, three_parts(v))
    assert torch.equal(dx, dx[:1].expand(n, e))


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("n,e,v", SIZES)
def test_every_product_of_dw(n, e, v, tied):
    w = torch.zeros(e, v, device="cuda")
    x = torch.zeros(n, e, device="cuda")
    row = torch.arange(e, device="cuda") % n
    a = fine(e, 4)
    x[row, torch.arange(e, device="cuda")] = a
    t = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    dw = dl.LinearCrossEntropyLoss("sum").value_and_grad(x, laid_out(w, tied), t)[2]
    p = torch.full((e,), 1.0 / v, device="cuda")
    near(dw[:, 9], a, p, three_parts(v))
    keep = torch.arange(v, device="cuda") != 3
    assert torch.equal(dw[:, keep], dw[:, 9:10].expand(e, v - 1))


SMALL = 2.0 ** -29
LOST = 1280 * SMALL + 2.0 ** -22  # terms beside the large one, and a handful of roundings


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("words", [2 ** 15, 2 ** 16, 2 ** 17])
def test_one_accumulator_of_dx_sums_at_most_1280_words(words, tied):
    n, e = 40, 48
    w = torch.full((e, words), SMALL, device="cuda")
    w[:, 0], w[:, 5] = 1.0, 0.0
    t = torch.full((n,), 5, dtype=torch.int32, device="cuda")
    dx = dl.LinearCrossEntropyLoss("sum").value_and_grad(torch.zeros(n, e, device="cuda"), laid_out(w, tied), t)[1]
    want = (1 + (words - 2) * SMALL) / words
    assert float((dx.double() - want).abs().max()) <= LOST * want


@pytest.mark.parametrize("tied", [False, True])
def test_one_accumulator_of_dw_sums_at_most_1280_rows(tied):
    n, e, v = 2 ** 17, 32, 64
    x = torch.full((n, e), SMALL, device="cuda")
    x[0] = 1.0
    t = torch.full((n,), 5, dtype=torch.int32, device="cuda")
    w = laid_out(torch.zeros(e, v, device="cuda"), tied)
    dw = dl.LinearCrossEntropyLoss("sum").value_and_grad(x, w, t)[2]
    want = torch.full((e, v), (1 + (n - 1) * SMALL) / v, dtype=torch.float64, device="cuda")
    want[:, 5] *= 1 - v
    assert bool(((dw.double() - want).abs() <= LOST * want.abs()).all())


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("e", [2048, 16384, 50000])
def test_one_accumulator_of_the_logits_sums_at_most_1280_numbers(e, grad, tied):
    n, v = 40, 80
    x = torch.full((n, e), SMALL, device="cuda")
    x[:, 0] = 1.0
    w = torch.zeros(e, v, device="cuda")
    w[:, 7] = 64.0
    t = torch.full((n,), 3, dtype=torch.int32, device="cuda")
    f = dl.LinearCrossEntropyLoss()
    loss = f.value_and_grad(x, laid_out(w, tied), t)[0] if grad else f.forward(x, laid_out(w, tied), t)
    want = 64 * (1 + (e - 1) * SMALL)
    assert abs(float(loss) - want) <= LOST * want
