"""Embedding lookup with scale and its gradient by sorted tokens.

The lookup is one product in fp32 and one rounding to the table's type: off
by at most half a step of that type on top of fp32's.  A gradient element is
an fp32 sum of m terms (each partial sum rounded) and one product: its error
is at most (m + 1) * 2^-24 * scale * sum |dy|.  The reference adds the same
fp32 / bf16 inputs in 64 bits.
"""
import math

import pytest
import torch

import dlvk_b200 as dl
from dlvk_b200.ops import nn

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 2.0 ** -24
HALF = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8}


def exact_grad(ids, dy, V, scale, padding=None):
    ids, dy = ids.reshape(-1).long().cpu(), dy.reshape(-1, dy.shape[-1]).double().cpu()
    ok = (ids >= 0) & (ids < V)
    if padding is not None:
        ok &= ids != padding
    ref = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, ids[ok], dy[ok]) * scale
    mag = torch.zeros(V, dy.shape[1], dtype=torch.float64).index_add_(0, ids[ok], dy[ok].abs()) * abs(scale)
    m = torch.bincount(ids[ok], minlength=V).double()[:, None]
    return ref, (m + 2) * EPS * mag + 1e-40


def check_grad(ids, dy, V, scale=1.0, padding=None):
    got = nn.embedding_grad(ids, dy, V, scale=scale, padding_idx=padding)
    ref, lim = exact_grad(ids, dy, V, scale, padding)
    assert got.dtype == torch.float32 and got.shape == ref.shape
    assert bool(((got.double().cpu() - ref).abs() <= lim).all())
    start = torch.randn(V, dy.shape[-1], device=dy.device)
    acc = start.clone()
    nn.embedding_grad(ids, dy, V, scale=scale, padding_idx=padding, out=acc, accumulate=True)
    lim = lim + 2 * EPS * start.abs().double().cpu()
    assert bool(((acc.double().cpu() - start.double().cpu() - ref).abs() <= lim).all())
    untouched = torch.bincount(ids.reshape(-1).clamp(-1, V).long().cpu() + 1, minlength=V + 2)[1:V + 1] == 0
    assert torch.equal(acc.cpu()[untouched], start.cpu()[untouched])
    return got


def zipf(n, V, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.multinomial(1.0 / (torch.arange(V) + 2.7), n, replacement=True, generator=g).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [1, 3, 8, 31, 64, 257, 1024, 2056])
@pytest.mark.parametrize("scale", [1.0, 0.37])
def test_lookup(device, dtype, D, scale):
    V = 77
    table = torch.randn(V, D, generator=torch.Generator().manual_seed(D)).to(dtype).to(device)
    ids = torch.tensor([[0, 76, 5], [5, -1, 77], [2 ** 31 - 1, -2 ** 31, 1]], device=device)
    for t in (torch.int32, torch.int64):
        got = nn.embedding_lookup(ids.to(t), table, scale=scale)
        ok = (ids >= 0) & (ids < V)
        ref = table[ids.clamp(0, V - 1)].double() * scale * ok[..., None]
        assert got.dtype == dtype and got.shape == ref.shape
        assert bool(((got.double() - ref).abs() <= ref.abs() * (HALF[dtype] + 2 * EPS)).all())
        if scale == 1.0:
            assert torch.equal(got, (table[ids.clamp(0, V - 1)] * ok[..., None]).to(dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_lookup_views_and_edges(device):
    base = torch.randn(20, 64, device=device)
    ids = torch.tensor([3, 19, 0], dtype=torch.int32, device=device)
    for table in (base[:, :24], base[:, 3:20], base[::2], base.t()[:20, ::3]):
        i = ids.clamp(max=table.shape[0] - 1)
        assert torch.equal(nn.embedding_lookup(i, table, scale=2.0), 2.0 * table[i.long()])
    strided = torch.arange(12, device=device).reshape(3, 4).t()
    assert torch.equal(nn.embedding_lookup(strided, base, scale=1.0), base[strided])
    assert nn.embedding_lookup(ids[:0], base).shape == (0, 64)
    assert nn.embedding_lookup(ids[0], base).shape == (64,)
    assert not nn.embedding_lookup(ids, base[:0]).any()
    assert nn.embedding_lookup(torch.tensor([2 ** 40 + 3, 3], device=device), base)[0].abs().sum() == 0


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 1000, 64), (2, 3, 5), (15, 40, 24), (16, 40, 24), (17, 1, 24),
                                   (100, 7, 1), (1000, 200, 40), (1024, 9, 1032), (1025, 5000, 8), (4099, 33, 130)])
def test_grad_sizes(device, dtype, n, V, D):
    ids = zipf(n, V, device)
    dy = torch.randn(n, D, generator=torch.Generator().manual_seed(n)).to(dtype).to(device)
    check_grad(ids.to(torch.int32), dy, V, scale=0.37)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,D", [(20000, 500, 48), (70000, 200000, 16), (70001, 3, 8), (3000, 152000, 33),
                                   (8192, 32000, 256)])
def test_grad_long(dtype, n, V, D):
    ids = zipf(n, V, "cuda")
    dy = torch.randn(n, D, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()
    check_grad(ids, dy, V, scale=2.0, padding=0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("count", [0, 1, 15, 16, 17, 31, 32, 33, 160])
def test_runs_that_end_at_chunk_borders(device, count):
    # word 1 has `count` tokens before word 2's begin: every place of a run's end
    ids = torch.tensor([1] * count + [2] * 40 + [4] * (64 - count % 32), device=device)
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1)).to(device)]
    dy = torch.randn(ids.numel(), 12, generator=torch.Generator().manual_seed(2)).to(device)
    check_grad(ids, dy, 6)


@pytest.mark.parametrize("device", DEVICES)
def test_grad_outside_padding_empty(device):
    ids = torch.tensor([[0, 4, 9], [-1, 10, 4], [2 ** 31 - 1, -2 ** 31, 0]], dtype=torch.int32, device=device)
    dy = torch.randn(3, 3, 20, device=device)
    dy[1, 0] = math.nan  # a position that counts nowhere
    dy[2, 1] = math.inf
    check_grad(ids, dy.nan_to_num(0, 0, 0), 10)
    got = nn.embedding_grad(ids, dy, 10)
    assert bool(torch.isfinite(got).all())
    got = check_grad(ids, dy.nan_to_num(0, 0, 0), 10, padding=4)
    assert not got[4].any()
    assert not nn.embedding_grad(torch.full((5,), 3, device=device), torch.ones(5, 8, device=device), 4,
                                 padding_idx=3).any()
    assert not nn.embedding_grad(ids[:0], dy[:0], 10).any()
    keep = torch.ones(10, 20, device=device)
    nn.embedding_grad(ids[:0], dy[:0], 10, out=keep, accumulate=True)
    assert torch.equal(keep, torch.ones(10, 20, device=device))
    assert nn.embedding_grad(ids, dy, 0).shape == (0, 20)


@pytest.mark.parametrize("device", DEVICES)
def test_grad_strided_and_broadcast_dy(device):
    ids = zipf(50, 9, device)
    base = torch.randn(50, 80, device=device)
    for dy in (base[:, :24], base[:, 3:20], torch.randn(24, 50, device=device).t(), base[:1, :24].expand(50, 24),
               base[:, :1].expand(50, 24)):
        check_grad(ids, dy, 9)
    check_grad(ids.reshape(5, 10).t(), base[:, :24].reshape(10, 5, 24), 9)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    ids, table, dy = torch.zeros(3, dtype=torch.int32, device=device), torch.zeros(4, 8, device=device), \
        torch.zeros(3, 8, device=device)
    E = (ValueError, RuntimeError)
    with pytest.raises(E):
        nn.embedding_lookup(ids.float(), table)
    with pytest.raises(E):
        nn.embedding_grad(ids.to(torch.int16), dy, 4)
    with pytest.raises(E):
        nn.embedding_grad(ids[:2], dy, 4)
    with pytest.raises(E):
        nn.embedding_grad(ids, dy, 4, accumulate=True)
    for out in (torch.zeros(4, 7, device=device), torch.zeros(4, 8, device=device, dtype=torch.float64)):
        with pytest.raises(E):
            nn.embedding_grad(ids, dy, 4, out=out)
    for pad in (-1, 4):
        with pytest.raises(ValueError):
            nn.embedding_grad(ids, dy, 4, padding_idx=pad)
        with pytest.raises(ValueError):
            dl.EmbeddingLayer(4, 8, padding_idx=pad)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    ids, table = torch.zeros(3, dtype=torch.int32), torch.zeros(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="ids on"):
        nn.embedding_lookup(ids, table)
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        nn.embedding_lookup(ids.cuda(), table.half())
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        nn.embedding_grad(ids.cuda(), torch.zeros(3, 8, device="cuda", dtype=torch.float64), 4)


@pytest.mark.gpu
def test_refusal_of_an_output_on_the_input():
    ids, dy = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 8, device="cuda")
    with pytest.raises(RuntimeError, match="memory"):
        nn.embedding_grad(ids, dy, 3, out=dy)


@pytest.mark.gpu
def test_same_bits_every_time():
    ids = zipf(8192, 3000, "cuda")
    dy = torch.randn(8192, 512, device="cuda").bfloat16()
    first = nn.embedding_grad(ids, dy, 3000, scale=3.0)
    for _ in range(10):
        assert torch.equal(nn.embedding_grad(ids, dy, 3000, scale=3.0), first)
    # a captured call gives the eager call's bits, also for other ids than it was captured with
    other = zipf(8192, 3000, "cuda", seed=5)
    want = nn.embedding_grad(other, dy, 3000, scale=3.0)
    g = torch.cuda.CUDAGraph()
    static = ids.clone()
    with torch.cuda.graph(g):
        out = nn.embedding_grad(static, dy, 3000, scale=3.0)
    g.replay()
    assert torch.equal(out, first)
    static.copy_(other)
    g.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layer_and_model(device, dtype):
    """The layer's gradient, scaled and without the padding word, by the formula;
    a second backward adds to the first."""
    from dlvk_b200.models.sequential import Sequential

    m = Sequential(device if device == "cpu" else "cuda:0", dtype, seed=0)
    m.add_embedding(50, 16, embed_scale=4.0, padding_idx=3)
    m.build()
    ids = torch.tensor([[1, 3, 7, 1], [3, 7, 7, 49]], dtype=torch.int32, device=device)
    W = m.m_layers[0].weight
    y = m.forward(ids)
    assert torch.equal(y, (W.value[ids.long()].float() * 4.0).to(y.dtype))
    gy = torch.randn(y.shape, device=device).to(y.dtype)
    ref, lim = exact_grad(ids, gy, 50, 4.0, 3)
    m.backward(gy)
    assert bool(((W.grad.double().cpu() - ref).abs() <= lim).all()) and not W.grad[3].any()
    m.forward(ids)
    m.backward(gy)
    assert bool(((W.grad.double().cpu() - 2 * ref).abs() <= 3 * lim).all())


def test_gradient_against_differences():
    """d sum(y * r) / dT by central differences of the fp32 lookup: it is linear, so
    the difference is exact up to the roundings of y (2^-24 |y| each, over h)."""
    g = torch.Generator().manual_seed(0)
    table, r = torch.randn(6, 5, generator=g), torch.randn(9, 5, generator=g)
    ids = torch.tensor([0, 1, 1, 5, 4, 1, 0, 5, 1])
    got = nn.embedding_grad(ids, r, 6, scale=0.7)
    h = 0.5
    for v in range(6):
        for d in range(5):
            up, dn = table.clone(), table.clone()
            up[v, d] += h
            dn[v, d] -= h
            diff = (nn.embedding_lookup(ids, up, 0.7) - nn.embedding_lookup(ids, dn, 0.7)).double() * r.double()
            lim = (4 * EPS * 0.7 * (table.abs().max() + h) * r.abs().sum()) / (2 * h) + 10 * EPS * r.abs().sum()
            assert abs(float(diff.sum()) / (2 * h) - float(got[v, d])) <= float(lim)


def test_architecture_keeps_scale_and_padding():
    from dlvk_b200.models.builder import model_from_architecture
    from dlvk_b200.models.sequential import Sequential

    m = Sequential("cpu", "fp32", seed=0)
    m.add_embedding(9, 4, embed_scale=2.0, padding_idx=1)
    m.build()
    c = model_from_architecture(m.architecture(), "cpu").m_layers[0]
    assert (c.embed_scale, c.padding_idx) == (2.0, 1)
    plain = Sequential("cpu", "fp32", seed=0)
    plain.add_embedding(9, 4)
    assert "embed_scale" not in plain.architecture()[0] and "padding_idx" not in plain.architecture()[0]
    k = m.clone().build().m_layers[0]
    assert (k.embed_scale, k.padding_idx) == (2.0, 1)


def test_onnx_export_keeps_the_scale(tmp_path):
    from dlvk_b200.export import onnx as ox
    from dlvk_b200.models.sequential import Sequential

    m = Sequential("cpu", "fp32", seed=0)
    m.add_embedding(9, 4, embed_scale=2.5)
    m.build()
    m.set_training(False)
    ids = torch.tensor([[1, 8, 0]])
    ox.export_model(m, str(tmp_path / "m.onnx"), [1, 3])
    got = ox.run(ox.parse_model((tmp_path / "m.onnx").read_bytes()), ids)
    assert torch.allclose(got, m.forward(ids), rtol=1e-6)
