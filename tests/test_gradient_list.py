"""GradientClipping.global_norm / clip_global_norm: a list of tensors as one
norm, against 64-bit sums.

Tolerances: the norm is one fp32 rounding (2^-24) of a sum kept in 64 bits,
whose terms are sums of four fp32 squares (each off by at most 3 * 2^-24, so
the root by half that): below 3 * 2^-24 together.  A scaled element adds the
coefficient's rounding and the product's: 2 * 2^-24 on top of the norm's 64-bit
error, and half a step of the output type.
"""
import math

import pytest
import torch

import dlvk_b200 as dl

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def exact_norm(ts):
    return math.sqrt(sum(float(t.detach().double().cpu().square().sum()) for t in ts))


def make(device, shapes, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to(dtype).to(device) for s in shapes]


def check_clip(grads, max_norm, out=None):
    before = [t.detach().clone() for t in grads]
    norm = dl.GradientClipping.clip_global_norm(grads, max_norm, out=out)
    want = exact_norm(before)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 3 * EPS * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for b, o in zip(before, grads if out is None else out):
        ref = b.double() * coef
        lim = ref.abs() * (3 * EPS + HALF[o.dtype]) + 2.0 ** -149
        assert bool(((o.double() - ref).abs() <= lim).all())
    if out is not None:
        assert all(torch.equal(b, t) for b, t in zip(before, grads))
    return norm


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes", [[(1,)], [(3,), (5, 7), ()], [(8192,), (8193,), (16385,), (4,)], [(1, 1)] * 70,
                                    [(127, 129), (64, 64, 3), (100001,)]])
def test_norm_and_clip(device, dtype, shapes):
    ts = make(device, shapes, dtype)
    want = exact_norm(ts)
    got = dl.GradientClipping.global_norm(ts)
    assert abs(float(got) - want) <= 3 * EPS * want
    check_clip([t.clone() for t in ts], 0.37 * want)
    check_clip([t.clone() for t in ts], 2.0 * want)
    check_clip(ts, 0.5 * want, out=[torch.full_like(t, 7.0, dtype=torch.float32) for t in ts])
    check_clip(ts, 0.5 * want, out=[torch.full_like(t, 7.0, dtype=torch.bfloat16) for t in ts])


@pytest.mark.parametrize("device", DEVICES)
def test_more_tensors_than_one_launch_holds(device):
    ts = make(device, [(1 + i % 9,) for i in range(2100)])
    check_clip(ts, 0.1)


@pytest.mark.parametrize("device", DEVICES)
def test_mixed_types_and_odd_places(device):
    flat = make(device, [(5000,)])[0]
    half = make(device, [(5000,)], torch.bfloat16, seed=1)[0]
    guard = flat.clone(), half.clone()
    ts, used = [], torch.zeros(5000, dtype=torch.bool, device=device)
    at = 1
    for n in (1, 2, 3, 5, 8, 13, 300, 1001, 2):
        ts += [flat[at:at + n], half[at:at + n]]
        used[at:at + n] = True
        at += n + 1
    check_clip(ts, 0.5)
    # nothing beside the views was written
    assert torch.equal(flat[~used], guard[0][~used]) and torch.equal(half[~used], guard[1][~used])


@pytest.mark.parametrize("device", DEVICES)
def test_strided_tensors(device):
    base = make(device, [(37, 3 * 24)])[0]
    keep = base.clone()
    parts = [base[:, :24], base[:, 24:48]]  # two column slices of one matrix, in place
    check_clip(parts + [make(device, [(19, 11)], seed=2)[0].t()], 0.25)
    assert torch.equal(base[:, 48:], keep[:, 48:])
    cube = make(device, [(4, 6, 10)], seed=3)[0]
    check_clip([cube.permute(2, 0, 1)[::2]], 0.25)
    src = make(device, [(6, 10)], seed=4)[0]
    check_clip([src.t()], 0.25, out=[torch.zeros(10, 6, device=device)])
    check_clip([src[:1].expand(5, 10)], 0.25, out=[torch.zeros(5, 10, device=device)])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e-10, 1e18, 3e25, 1e38])
def test_range_of_fp32(device, size):
    # squares of these leave fp32; their norm does not (1e38 * sqrt(9) < 3.4e38)
    ts = [torch.full((4,), size, device=device), torch.tensor([size, 0.0, size, size, 0.0, size, size], device=device)]
    want = exact_norm(ts)
    assert abs(float(dl.GradientClipping.global_norm(ts)) - want) <= 3 * EPS * want


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", [0, 3, 9000])
def test_not_finite_scales_nothing(device, bad, where):
    ts = make(device, [(5,), (9001,)])
    ts[1][where] = bad
    before = [t.clone() for t in ts]
    norm = float(dl.GradientClipping.clip_global_norm(ts, 0.1))
    assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
    assert all(torch.equal(a.nan_to_num(9.0, 8.0, 7.0), b.nan_to_num(9.0, 8.0, 7.0)) for a, b in zip(before, ts))
    out = [torch.zeros_like(t) for t in ts]
    dl.GradientClipping.clip_global_norm(ts, 0.1, out=out)
    assert torch.equal(out[0], ts[0])


@pytest.mark.parametrize("device", DEVICES)
def test_zero_empty_and_repeated(device):
    z = [torch.zeros(10, device=device), torch.zeros(0, 4, device=device)]
    assert float(dl.GradientClipping.clip_global_norm(z, 1.0)) == 0.0 and not z[0].any()
    assert float(dl.GradientClipping.global_norm(z[1:])) == 0.0
    assert float(dl.GradientClipping.clip_global_norm(z[1:], 1.0)) == 0.0
    assert float(dl.GradientClipping.global_norm([])) == 0.0
    t = make(device, [(100,)])[0]
    assert abs(float(dl.GradientClipping.global_norm([t, t])) - math.sqrt(2) * exact_norm([t])) < 1e-5
    assert float(dl.GradientClipping.global_norm(x for x in [t])) == float(dl.GradientClipping.global_norm([t]))


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    t = make(device, [(8,)])[0]
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError):
            dl.GradientClipping.clip_global_norm([t], bad)
    with pytest.raises(ValueError):
        dl.GradientClipping.clip_global_norm([t], 1.0, out=[])
    with pytest.raises((ValueError, RuntimeError)):
        dl.GradientClipping.clip_global_norm([t], 1.0, out=[torch.zeros(7, device=device)])
    with pytest.raises((ValueError, RuntimeError)):
        dl.GradientClipping.global_norm([t, t.double()])


@pytest.mark.gpu
def test_refusals_of_shared_memory():
    clip = dl.GradientClipping.clip_global_norm
    t = make("cuda", [(64,)])[0]
    before = t.clone()
    m = make("cuda", [(8, 24)])[0]
    for bad in ([t, t], [t[:40], t[32:]], [m[:, :9], m[:, 8:16]], [m, m[:, 3:5]], [t[:1].expand(4)]):
        with pytest.raises(RuntimeError, match="share memory|repeats"):
            clip(bad, 0.1)
    with pytest.raises(RuntimeError, match="share memory"):
        clip([t[:32]], 0.1, out=[t[16:48]])
    with pytest.raises(RuntimeError, match="another device"):
        clip([t, torch.zeros(4)], 0.1)
    with pytest.raises(RuntimeError, match="neither"):
        clip([t, torch.zeros(4, device="cuda", dtype=torch.float16)], 0.1)
    with pytest.raises(RuntimeError, match="strides"):
        clip([torch.zeros(2, 2, 2, 2, 2, 16, device="cuda")[..., ::2].permute(4, 2, 0, 3, 1, 5)], 0.1)
    assert torch.equal(t, before)


@pytest.mark.parametrize("device", DEVICES)
def test_inputs_that_share_memory_are_only_read(device):
    g = make(device, [(12, 40)])[0]
    grads = [g, g[:, 8:24], g, g[3:5]]
    out = [torch.empty(t.shape, device=device) for t in grads]
    want = torch.cat([t.double().reshape(-1) for t in grads]).norm()
    norm = dl.GradientClipping.clip_global_norm(grads, 0.5, out=out)
    assert float(norm) == pytest.approx(float(want), rel=1e-6)
    for t, o in zip(grads, out):  # two fp32 roundings: the factor's and the product's
        assert bool(((o.double() - t.double() * 0.5 / (want + 1e-6)).abs() <= 3 * 2.0 ** -24 * t.double().abs()).all())


@pytest.mark.gpu
def test_refusal_of_an_output_on_another_input():
    flat = torch.zeros(4096, device="cuda")
    clip = dl.GradientClipping.clip_global_norm
    outs = [flat[i * 512:(i + 1) * 512] for i in range(8)]
    grads = [torch.ones(512, device="cuda") for _ in range(8)]
    clip(grads, 1.0, out=outs)
    clip(grads, 1.0, out=outs[::-1])
    for k, bad in ((0, flat[512:1024]), (3, flat[100:612]), (7, flat[3583:4095]), (5, flat[2600:3112])):
        with pytest.raises(RuntimeError, match="share memory"):
            clip(grads[:k] + [bad] + grads[k + 1:], 1.0, out=outs)
    m = torch.zeros(6, 40, device="cuda")
    cols = [m[:, 8 * i:8 * i + 8] for i in range(4)]
    clip([torch.ones(6, 8, device="cuda") for _ in cols], 1.0, out=cols)
    clip(cols + [m[:, 32:].clone()], 1.0, out=[torch.zeros(6, 8, device="cuda") for _ in cols] + [m[:, 32:]])
    with pytest.raises(RuntimeError, match="share memory"):
        clip(cols + [m[:, 30:38]], 1.0, out=[torch.zeros(6, 8, device="cuda") for _ in cols] + [m[:, 32:]])


@pytest.mark.gpu
def test_refusal_of_an_output_that_repeats_its_elements():
    t = make("cuda", [(64,)])[0]
    before = t.clone()
    clip = dl.GradientClipping.clip_global_norm
    for bad in (t.unfold(0, 8, 4), t.as_strided((4, 4), (1, 1)), t.as_strided((3, 5), (2, 1))):
        with pytest.raises(RuntimeError, match="repeats"):
            clip([bad], 0.1)
        with pytest.raises(RuntimeError, match="repeats"):
            clip([torch.ones(bad.shape, device="cuda")], 0.1, out=[bad])
    assert torch.equal(t, before)
    # read, they count what they show
    norm = float(dl.GradientClipping.global_norm([t.unfold(0, 8, 4)]))
    assert norm == pytest.approx(float(before.unfold(0, 8, 4).double().square().sum().sqrt()), rel=1e-6)


@pytest.mark.gpu
def test_captured_and_repeated_bits():
    ts = make("cuda", [(70001,), (333, 77), (5,)])
    out = [torch.zeros_like(t) for t in ts]
    eager = dl.GradientClipping.clip_global_norm(ts, 0.5, out=out)
    want = [o.clone() for o in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        dl.GradientClipping.clip_global_norm(ts, 0.5, out=out)
        with torch.cuda.graph(g, stream=side):
            norm = dl.GradientClipping.clip_global_norm(ts, 0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for o in out:
        o.zero_()
    g.replay()
    assert torch.equal(norm, eager) and all(torch.equal(a, b) for a, b in zip(out, want))
    for t in ts:
        t.mul_(3.0)
    g.replay()
    assert abs(float(norm) / float(eager) - 3.0) < 1e-6


@pytest.mark.gpu
def test_on_a_side_stream_after_its_producer():
    side = torch.cuda.Stream()
    x = torch.zeros(1 << 20, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            x.add_(1.0)
        norm = dl.GradientClipping.clip_global_norm([x], 1.0)
    side.synchronize()
    assert abs(float(norm) - 20.0 * 1024.0) <= 3 * EPS * 20480.0
