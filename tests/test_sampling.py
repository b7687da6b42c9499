"""The choice of the next word: every answer against the rule, written out one
word at a time in Python's numbers (64 bits; sums by math.fsum).

Answers are whole numbers.  A rule in 64 bits and sums in steps of 2^-44 can
part only where a running sum lies within 2^-26 (2^18 words, half a step each)
of a border relative to the total; the uniform numbers of the random tests are
taken so that none does (`safe`)."""
import math

import pytest
import torch

from dlvk_b200.ops import sampling

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.bfloat16]
NEAR = 2.0 ** -26


def kept_words(z, temperature, top_k, top_p, min_p):
    """({word: weight} that is left, whether a border was too near to tell)."""
    z = [-math.inf if math.isnan(v) else v for v in z]
    top = max(z)
    if top == -math.inf:
        return {}, False
    order = sorted(range(len(z)), key=lambda i: (-z[i], i))
    if not temperature > 0:
        return {order[0]: 1.0}, False
    weight = lambda v: 1.0 if v == top else 0.0 if top == math.inf else math.exp((v - top) / temperature)  # noqa: E731
    if top_k > 0:
        order = order[:top_k]
    total = math.fsum(weight(z[i]) for i in order)
    kept, upto, close = {}, [], False
    run = 0.0
    for place, i in enumerate(order):
        w = weight(z[i])
        if top_p < 1 and place > 0:
            near = abs(run - top_p * total) <= NEAR * total
            # equal weights add up exactly alike on both sides: not a question of rounding
            close = close or (near and run != top_p * total)
            if run >= top_p * total:
                break
        run += w
        if w >= min_p:
            kept[i] = w
        close = close or (min_p > 0 and abs(w - min_p) <= NEAR and w != min_p)
    return kept, close


def word_of(kept, u):
    """(the word, whether u is too near a border)."""
    if not kept:
        return -1, False
    total, run = math.fsum(kept.values()), 0.0
    for i in sorted(kept):
        run += kept[i]
        if run > u * total:
            return i, abs(run - u * total) <= NEAR * total or abs(run - kept[i] - u * total) <= NEAR * total and u > 0
    return max(kept), True


def check(logits, settings, device, seed=0, draws=6, **as_given):
    """Some uniform numbers for every row, away from the borders."""
    rows = logits.shape[0]
    g = torch.Generator().manual_seed(seed)
    per_row = [{k: (v[r].item() if torch.is_tensor(v) else v) for k, v in settings.items()} for r in range(rows)]
    left = [kept_words(logits[r].double().tolist(), **per_row[r]) for r in range(rows)]
    given = {k: v.to(device) if torch.is_tensor(v) else v for k, v in settings.items()}
    for _ in range(draws):
        u = torch.rand(rows, generator=g)
        got = sampling.sample_tokens(logits.to(device), u.to(device), **given)
        assert got.dtype == torch.int32 and got.shape == (rows,)
        for r, token in enumerate(got.tolist()):
            want, close = word_of(left[r][0], float(u[r]))
            if not close and not left[r][1]:
                assert token == want, (r, token, want, per_row[r])


def rows_of(n, words, dtype, seed=0, spread=3.0):
    return (torch.randn(n, words, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


PLAIN = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("words", [1, 2, 31, 33, 257, 1023, 1025, 4097, 9000])
def test_sizes(device, dtype, words):
    z = rows_of(3, words, dtype, words)
    check(z, PLAIN, device, words)
    check(z, dict(temperature=0.7, top_k=5, top_p=0.9, min_p=0.02), device, words)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("setting", [dict(temperature=0.3), dict(temperature=5.0), dict(top_k=1), dict(top_k=2), dict(top_k=50),
                                     dict(top_k=600), dict(top_k=10 ** 9), dict(top_p=0.1), dict(top_p=0.5), dict(top_p=0.999),
                                     dict(top_p=1e-9), dict(min_p=0.3), dict(min_p=1.0), dict(top_k=40, top_p=0.8),
                                     dict(temperature=1.4, top_k=300, top_p=0.95, min_p=0.001), dict(top_p=0.7, min_p=0.2)])
def test_settings(device, dtype, setting):
    check(rows_of(4, 601, dtype, 3), dict(PLAIN, **setting), device, 1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_settings_of_each_row(device, dtype):
    z = rows_of(12, 900, dtype, 5)
    check(z, dict(temperature=torch.tensor([0.0, 0.5, 1.0, 2.0] * 3), top_k=torch.tensor([0, 1, 30, 2000, -4, 7] * 2, dtype=torch.int32),
                  top_p=torch.tensor([1.0, 0.5, 0.9] * 4), min_p=torch.tensor([0.0, 0.05] * 6)), device, 2)
    check(z, dict(PLAIN, top_p=torch.tensor([0.25, 0.5, 0.75, 1.0] * 3)), device, 3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_go_by_their_numbers(device, dtype):
    """Whole numbers of equal weights: every border is exact."""
    words = 1000
    z = torch.zeros(1, words, dtype=dtype, device=device)
    one = lambda u, **kw: int(sampling.sample_tokens(z, torch.tensor([u], device=device), **kw))  # noqa: E731
    assert one(0.0) == 0 and one(0.5) == 500 and one(1 - 2.0 ** -24) == 999
    assert one(0.0, temperature=0.0) == 0
    assert one(0.75, top_k=4) == 3 and one(0.999, top_k=1) == 0
    assert one(1 - 2.0 ** -24, top_p=0.25) == 249 and one(1 - 2.0 ** -24, top_p=0.2501) == 250
    assert one(1 - 2.0 ** -24, top_k=100, top_p=0.5) == 49
    assert one(1 - 2.0 ** -24, min_p=1.0) == 999
    z[0, 700:] = 1.0  # larger ones last
    assert one(0.0, temperature=0.0) == 700 and one(0.0, top_k=300) == 700 and one(0.0, top_k=301) == 0
    assert one(1 - 2.0 ** -24, top_k=17) == 716 and one(1 - 2.0 ** -24, min_p=0.9) == 999
    few = torch.tensor([[0.0, -0.0, 0.0]], dtype=dtype, device=device)
    assert int(sampling.sample_tokens(few, torch.tensor([0.9], device=device), top_k=2)) == 1
    assert int(sampling.sample_tokens(few, torch.tensor([0.9], device=device), temperature=0.0)) == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_masks_infinities_and_nan(device, dtype):
    low = torch.finfo(dtype).min
    z = rows_of(8, 300, dtype, 7)
    z[0] = -math.inf
    z[1, :299] = -math.inf
    z[2, 10:] = low
    z[3, ::2] = math.nan
    z[4, 5], z[4, 200] = math.inf, math.inf
    z[5] = math.nan
    z[6] = low
    z[7, 3:] = -math.inf
    for s in (PLAIN, dict(PLAIN, temperature=0.0), dict(PLAIN, top_k=20), dict(PLAIN, top_p=0.6),
              dict(PLAIN, min_p=0.1), dict(temperature=0.5, top_k=7, top_p=0.9, min_p=0.01)):
        check(z, s, device, 4)
        got = sampling.sample_tokens(z.to(device), torch.full((8,), 0.3, device=device), **s)
        assert got[0] == -1 and got[5] == -1 and got[1] == 299 and got[2] < 10 and got[4] in (5, 200) and got[7] < 3


@pytest.mark.parametrize("device", DEVICES)
def test_uniform_numbers_and_settings_outside_their_ranges(device):
    z = rows_of(1, 64, torch.float32, 9)
    call = lambda u, **kw: int(sampling.sample_tokens(z.to(device), torch.tensor([u], device=device), **kw))  # noqa: E731
    assert call(-1.0) == 0 and call(math.nan) == 0 and call(1.0) == 63 and call(7.0) == 63
    best = int(z.argmax())
    assert call(0.5, temperature=-1.0) == best and call(0.5, temperature=math.nan) == best
    assert call(0.9, top_p=0.0) == best and call(0.9, top_p=-2.0) == best and call(0.9, min_p=3.0) == best
    assert call(0.4, top_p=math.nan, min_p=math.nan) == call(0.4) == call(0.4, top_p=2.0, min_p=-1.0, top_k=-5)
    wide = torch.full((1, 64), 1e38)
    wide[0, 7], wide[0, 9] = 3e38, -3e38
    got = sampling.sample_tokens(wide.to(device), torch.tensor([0.99], device=device), temperature=0.5)
    assert int(got) == 7


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_and_shapes(device, dtype):
    z = rows_of(6, 120, dtype, 11).to(device)
    u = torch.rand(6, generator=torch.Generator().manual_seed(1)).to(device)
    want = sampling.sample_tokens(z, u, top_k=9)
    base = torch.zeros(6, 131, dtype=dtype, device=device)
    base[:, 5:125] = z
    assert torch.equal(sampling.sample_tokens(base[:, 5:125], u, top_k=9), want)
    assert torch.equal(sampling.sample_tokens(z.t().contiguous().t(), u, top_k=9), want)
    assert torch.equal(sampling.sample_tokens(z.reshape(2, 3, 120), u.reshape(2, 3), top_k=9), want.reshape(2, 3))
    assert torch.equal(sampling.sample_tokens(z[0], u[0], top_k=9), want[0])
    same = sampling.sample_tokens(z[:1].expand(6, 120), u[:1].expand(6), top_k=9)
    assert bool((same == want[0]).all())
    assert sampling.sample_tokens(z[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    z, u = torch.zeros(2, 5, device=device), torch.zeros(2, device=device)
    for call in (lambda: sampling.sample_tokens(z.half(), u), lambda: sampling.sample_tokens(z[:, :0], u),
                 lambda: sampling.sample_tokens(z, u[:1]), lambda: sampling.sample_tokens(z, u.double()),
                 lambda: sampling.sample_tokens(z, u, top_k=torch.ones(2, device=device)),
                 lambda: sampling.sample_tokens(z, u, temperature=torch.ones(3, device=device)),
                 lambda: sampling.sample_tokens(z, u, top_p=torch.ones(2, dtype=torch.float64, device=device)),
                 lambda: sampling.sample_tokens(torch.zeros(1, 2 ** 18 + 1, device=device), u[:1])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_refusals_of_devices():
    z, u = torch.zeros(2, 5, device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError):
        sampling.sample_tokens(z, u.cpu())
    with pytest.raises(ValueError):
        sampling.sample_tokens(z, u, top_p=torch.ones(2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,words", [(1, 50257), (3, 128000), (40, 32000), (200, 1999), (2, 2 ** 18)])
def test_large_against_the_cpu(dtype, rows, words):
    """The CPU's path makes the same whole numbers, so even borders agree; its
    weights differ from the kernel's by an exponential's last bit of 53, which
    reaches a step of 2^-44 for one word in 2^8 and a border for none of these."""
    z = rows_of(rows, words, dtype, words, 2.5)
    z[0, : words // 2] = -math.inf
    u = torch.rand(rows, generator=torch.Generator().manual_seed(3))
    for s in (PLAIN, dict(PLAIN, top_k=50, top_p=0.95, temperature=0.8), dict(PLAIN, top_p=0.9), dict(PLAIN, top_k=3000),
              dict(PLAIN, min_p=0.05), dict(PLAIN, temperature=0.0)):
        want = sampling.sample_tokens(z, u, **s)
        got = sampling.sample_tokens(z.cuda(), u.cuda(), **s)
        assert torch.equal(got.cpu(), want), s


@pytest.mark.gpu
def test_streams_and_graphs():
    z, u = rows_of(5, 3000, torch.float32, 1).cuda(), torch.rand(5).cuda()
    kw = dict(top_k=40, top_p=0.9, temperature=torch.full((5,), 0.8, device="cuda"))
    want = sampling.sample_tokens(z, u, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sampling.sample_tokens(z, u, **kw)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = sampling.sample_tokens(z, u, **kw)
        graphs.append((g, out))
    z.copy_(z.flip(0))
    want = sampling.sample_tokens(z, u, **kw)
    for _ in range(2):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out in graphs)


@pytest.mark.gpu
def test_shares_follow_the_weights():
    """Uniform numbers spread evenly give each word its share of them, to one number."""
    z = rows_of(1, 50, torch.float32, 2, 1.0).cuda()
    n = 20000
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float().cuda()
    got = torch.bincount(sampling.sample_tokens(z.expand(n, 50), u).long(), minlength=50).double()
    share = torch.softmax(z[0].double(), 0) * n
    assert bool(((got - share).abs() <= 1.01 + n * 2.0 ** -24).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature,spread", [(1e38, 1e38), (1e30, 1e30), (3e-30, 1e-30), (1e-300, 1.0), (1e300, 1.0),
                                                (math.inf, 1.0), (5e-324, 3.0)])
def test_temperatures_and_logits_at_the_ends_of_their_ranges(device, dtype, temperature, spread):
    """Differences of logits that overflow fp32 or vanish against the temperature."""
    z = rows_of(2, 6001, torch.float32, 9, 1.0).mul_(spread).clamp_(-3.2e38, 3.2e38).to(dtype)
    for s in (dict(top_p=0.9), dict(top_p=0.5, top_k=4000), dict(top_k=2500, min_p=0.01), dict(top_p=0.3)):
        check(z, dict(PLAIN, **s, temperature=temperature), device, 3, draws=2)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("words", [1100, 1600, 40000])
def test_cuts_in_runs_of_equal_logits(device, words):
    """One number, and two with ties across the cut: weights of 1 and 1/2 (to a
    part of 2^-53) add up without a border within 2^-26 of these shares."""
    z = torch.zeros(3, words)
    z[1, ::2] = math.log(0.5)
    z[2, words // 3:] = math.log(0.5)
    for s in (dict(top_p=0.30001), dict(top_p=0.99999), dict(top_p=1 - 2.0 ** -50), dict(top_k=words // 2 + 7),
              dict(top_k=1152), dict(top_k=1153), dict(top_k=1536), dict(top_k=1537), dict(top_k=words - 1),
              dict(top_k=words - 3, top_p=0.70003), dict(min_p=0.6, top_p=0.8003)):
        check(z, dict(PLAIN, **s), device, 5, draws=2)


@pytest.mark.gpu
def test_weights_of_a_few_steps():
    """200000 words that weigh two steps of 2^-44 each behind one of 2^44: shares
    that end among them, against the CPU's same whole numbers."""
    z = torch.full((2, 200001), -30.0)
    z[0, 7], z[1, 200000] = 0.0, 0.0
    for p in (1 - 1e-8, 1 - 2e-8, 1 - 1e-9, 1 - 1e-12, 0.5):
        for u in (0.0, 0.999, 1 - 2.0 ** -24):
            u = torch.full((2,), u)
            want = sampling.sample_tokens(z, u, top_p=p)
            assert torch.equal(sampling.sample_tokens(z.cuda(), u.cuda(), top_p=p).cpu(), want)


@pytest.mark.gpu
def test_rows_past_31_bits():
    z = torch.empty(70000, 32000, dtype=torch.bfloat16, device="cuda")
    z.normal_(generator=torch.Generator("cuda").manual_seed(1))
    u = torch.rand(70000, device="cuda")
    got = sampling.sample_tokens(z, u, top_k=50, top_p=0.9)
    for part in (slice(0, 300), slice(67100, 67120), slice(69700, 70000)):
        assert torch.equal(got[part], sampling.sample_tokens(z[part].clone(), u[part], top_k=50, top_p=0.9))


@pytest.mark.parametrize("device", DEVICES)
def test_logits_that_are_no_normal_numbers(device):
    """Logits of some steps of 2^-149 and temperatures as small, where 1 / temperature is no number of fp32."""
    z = torch.randint(0, 200, (2, 6001), generator=torch.Generator().manual_seed(4)).float() * 2.0 ** -149
    for t in (2.0 ** -125, 2.0 ** -140, 2.0 ** -149, 1e-30):
        for s in (dict(top_p=0.9), dict(top_k=2500), dict(top_p=0.4, top_k=3999)):
            check(z, dict(PLAIN, **s, temperature=t), device, 4, draws=2)
