"""StateSpaceLayer and Sequential.generate: the layer's output and gradients
against its formula in 64 bits, pieces and single tokens, a training step, and
text written token by token."""
import math

import pytest
import torch

import dlvk_b200 as dl
from dlvk_b200.export import onnx
from dlvk_b200.models import zoo
from dlvk_b200.models.builder import model_from_architecture
from dlvk_b200.models.sequential import Sequential
from dlvk_b200.ops import sampling

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def layer_ref(layer, x):
    """The layer's formula in 64 bits with autograd; returns (output, {name: leaf})."""
    p = {k: getattr(layer, k).value.detach().cpu().double().requires_grad_(True)
         for k in ("w_in", "w_x", "w_dt", "w_out")}
    for k in ("conv_weight", "conv_bias", "dt_bias", "a_log", "skip"):
        p[k] = getattr(layer, k).master.detach().cpu().double().requires_grad_(True)
    B, T, _ = x.shape
    W, N, G, K = layer.width, layer.d_state, layer.groups, layer.d_conv
    xz = x @ p["w_in"]
    v, z = xz[..., :W], xz[..., W:]
    v = torch.cat([torch.zeros(B, K - 1, W, dtype=torch.float64), v], 1)
    v = sum(p["conv_weight"][:, j] * v[:, j:j + T] for j in range(K)) + p["conv_bias"]
    v = v * torch.sigmoid(v)
    low, b, c = (v @ p["w_x"]).split([layer.dt_rank, G * N, G * N], -1)
    b, c = (t.reshape(B, T, G, N).repeat_interleave(W // G, 2) for t in (b, c))
    step = torch.nn.functional.softplus(low @ p["w_dt"] + p["dt_bias"], threshold=1e9)
    h, ys = torch.zeros(B, W, N, dtype=torch.float64), []
    for t in range(T):
        h = torch.exp(step[:, t, :, None] * -torch.exp(p["a_log"])) * h + (step[:, t] * v[:, t])[..., None] * b[:, t]
        ys.append((h * c[:, t]).sum(-1) + p["skip"] * v[:, t])
    y = torch.stack(ys, 1) * z * torch.sigmoid(z)
    out = y @ p["w_out"]
    return out + x if layer.residual else out, p


def make(device, dtype, groups=1, residual=False, d_model=32, **kw):
    dl.manual_seed(3)
    layer = dl.StateSpaceLayer(d_model, groups=groups, residual=residual, **kw)
    layer.to(device, dtype)
    return layer


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("groups,residual,kw", [(1, False, {}), (2, True, dict(d_state=8, d_conv=3)), (1, True, dict(d_state=5, dt_rank=3))])
def test_layer_fp32(device, groups, residual, kw):
    """fp32: at most some 200 roundings of 2^-24 (3xTF32-like products 2^-17) on
    sums whose terms do not cancel by more than 2^6: 2^-10 of the largest value."""
    layer = make(device, torch.float32, groups, residual, **kw)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 19, 32, generator=g)
    dy = torch.randn(3, 19, 32, generator=g)
    y = layer.forward(x.to(device))
    dx = layer.backward(dy.to(device))
    xr = x.double().requires_grad_(True)
    ref, p = layer_ref(layer, xr)
    names = list(p)
    grads = torch.autograd.grad(ref, [xr] + [p[k] for k in names], dy.double())
    near = lambda a, b: bool(((a.cpu().double() - b).abs() <= 2.0 ** -10 * b.abs().max()).all())  # noqa: E731
    assert near(y, ref) and near(dx, grads[0])
    for k, r in zip(names, grads[1:]):
        assert near(getattr(layer, k).grad, r), k


@pytest.mark.gpu
def test_layer_bf16():
    """bf16: eight roundings of 2^-8 in a row from x to the output (24 with the
    way back), of values whose sums grow errors no more than themselves."""
    layer = make("cuda", torch.bfloat16, d_model=64, residual=True)
    g = torch.Generator().manual_seed(6)
    x, dy = (torch.randn(2, 70, 64, generator=g).bfloat16() for _ in range(2))
    y = layer.forward(x.cuda())
    dx = layer.backward(dy.cuda())
    xr = x.double().requires_grad_(True)
    ref, p = layer_ref(layer, xr)
    names = list(p)
    grads = torch.autograd.grad(ref, [xr] + [p[k] for k in names], dy.double())
    off = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())  # noqa: E731
    assert off(y, ref) <= 8 * 2.0 ** -8 and off(dx, grads[0]) <= 24 * 2.0 ** -8
    for k, r in zip(names, grads[1:]):
        assert off(getattr(layer, k).grad, r) <= 24 * 2.0 ** -8, k


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_accumulate(device):
    layer = make(device, torch.float32)
    x = torch.randn(2, 9, 32, device=device)
    dy = torch.randn(2, 9, 32, device=device)
    layer.forward(x)
    layer.backward(dy)
    once = {p.name: p.grad.clone() for p in layer.parameters()}
    layer.forward(x)
    torch.autograd.grad(layer._last_out, layer._last_in, dy)  # without zero_grad
    for p in layer.parameters():
        want = 2 * once[p.name]
        assert bool(((p.grad - want).abs() <= 2.0 ** -20 * want.abs().max() + 1e-30).all()), p.name


@pytest.mark.parametrize("device", DEVICES)
def test_prompt_pieces_steps_and_lengths(device):
    layer = make(device, torch.float32, groups=2, residual=True)
    layer.track = False
    x = torch.randn(3, 23, 32, generator=torch.Generator().manual_seed(1)).to(device)
    whole = layer.forward(x).detach()
    tol = 2.0 ** -16 * float(whole.abs().max())  # two orders of the same fp32 sums of up to 64 terms
    state, parts = None, []
    for a, e in ((0, 7), (7, 8), (8, 20)):
        y, state = layer.prompt(x[:, a:e], state)
        parts.append(y)
    for t in range(20, 23):
        parts.append(layer.step(x[:, t], state)[:, None])
    assert float((torch.cat(parts, 1) - whole).abs().max()) <= tol
    n = torch.tensor([23, 1, 10], dtype=torch.int32, device=device)
    y, state = layer.prompt(x, lengths=n)
    for i, k in enumerate(n.tolist()):
        yi, si = layer.prompt(x[i:i + 1, :k])
        assert float((y[i, :k] - yi[0]).abs().max()) <= tol
        assert torch.equal(state.conv[i], si.conv[0]) or float((state.conv[i] - si.conv[0]).abs().max()) <= tol
        assert float((state.scan[i] - si.scan[0]).abs().max()) <= 2.0 ** -16 * float(si.scan.abs().max())
    zero = layer.init_state(3)
    assert zero.conv.shape == state.conv.shape and zero.scan.shape == state.scan.shape
    assert torch.equal(layer.prompt(x, zero)[0], layer.prompt(x)[0])


def model(device, dtype, seed=0):
    m = Sequential(device, dtype, seed=seed)
    m.add_embedding(50, 32)
    m.add_layernorm(32)
    m.add_state_space(32, residual=True)
    m.add(dl.ResidualLayer(dl.StateSpaceLayer(32, d_state=8, groups=2)))
    m.add(dl.ResidualLayer(dl.DenseLayer(32, 32)))
    m.add_layernorm(32)
    m.add_dense(32, 50)
    m.add_softmax()
    return m.build()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_generate_is_the_model_run_again(device, dtype):
    """Every word is the choice from the whole model's logits of all tokens so
    far.  The two ways round differently, so the uniform numbers are moved
    off the borders: each word is checked where its choice does not change
    within the logits' error (2^-12 in fp32, 2^-4 in bf16, of logits about 1)."""
    m = model(device, dtype)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, 50, (4, 11), generator=g, dtype=torch.int32)
    n = [11, 4, 1, 9]
    u = torch.rand(4, 6, generator=g)
    got = m.generate(prompt, 6, u, lengths=n, temperature=0.9, top_k=20)
    assert got.dtype == torch.int32 and got.shape == (4, 6) and m.is_training
    err = 2.0 ** -12 if dtype == "fp32" else 2.0 ** -4
    m.set_training(False)
    told = 0
    for i in range(4):
        seq = prompt[i, :n[i]].tolist()
        for k in range(6):
            z = m.forward_logits(torch.tensor([seq], dtype=torch.int32)).detach()[:, -1].float().cpu()
            draws = [z + err * torch.randn(z.shape, generator=g) for _ in range(30)]
            words = {int(sampling.sample_tokens(d, u[i:i + 1, k], 0.9, 20)) for d in draws + [z]}
            assert int(got[i, k]) in words
            told += len(words) == 1
            seq.append(int(got[i, k]))
    assert told >= (18 if dtype == "fp32" else 4)


@pytest.mark.parametrize("device", DEVICES)
def test_generate_greedy_and_refusals(device):
    m = model(device, "fp32", seed=4)
    prompt = torch.randint(0, 50, (2, 5), generator=torch.Generator().manual_seed(3))
    a = m.generate(prompt, 4, temperature=0.0)
    assert torch.equal(a, m.generate(prompt, 4, temperature=0.0))
    assert m.generate(prompt, 0).shape == (2, 0)
    assert torch.equal(m.generate(prompt, 1, temperature=0.0), a[:, :1])
    for call in (lambda: m.generate(prompt[:, :0], 2), lambda: m.generate(prompt[0], 2),
                 lambda: m.generate(prompt, 2, lengths=[0, 5]), lambda: m.generate(prompt, 2, lengths=[6, 5]),
                 lambda: m.generate(prompt, 2, lengths=[5]), lambda: m.generate(prompt, 2, torch.rand(2, 3)),
                 lambda: zoo.transformer("cpu", "fp32", vocab=20, d_model=16, layers=1, heads=2, d_ff=16).generate(prompt, 2),
                 lambda: Sequential("cpu", "fp32").add_dense(4, 4).generate(prompt, 2)):
        with pytest.raises(ValueError):
            call()
    for bad in (dict(d_conv=1), dict(d_conv=5), dict(d_state=0), dict(d_state=65), dict(groups=5), dict(dt_rank=0)):
        with pytest.raises(ValueError):
            dl.StateSpaceLayer(32, **bad)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_training_steps_run(device, dtype):
    m = model(device, dtype)
    x = torch.randint(0, 50, (3, 12), dtype=torch.int32, device=device)
    y = torch.randint(0, 50, (3, 12), dtype=torch.int32, device=device)
    before = m.store.master.clone()
    for loss in (dl.CrossEntropyLoss(), dl.LinearCrossEntropyLoss()):
        value = m.train_step(x, y, loss, dl.Adam(1e-3))
        assert math.isfinite(float(value))
    assert bool(torch.isfinite(m.store.grad).all()) and not torch.equal(before, m.store.master)


@pytest.mark.gpu
def test_captured_training_step_is_the_eager_one():
    x = torch.randint(0, 50, (3, 40), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).cuda()
    y = x.roll(-1, 1).contiguous()
    a, b = model("cuda", "bf16"), model("cuda", "bf16")
    assert torch.equal(a.store.master, b.store.master)
    step = dl.TrainStep(a, dl.CrossEntropyLoss(), dl.Adam(1e-3))
    opt = dl.Adam(1e-3)
    for _ in range(4):
        step(x, y)
        b.train_step(x, y, dl.CrossEntropyLoss(), opt)
    torch.cuda.synchronize()
    assert torch.equal(a.store.master, b.store.master)


@pytest.mark.parametrize("device", DEVICES)
def test_saved_rebuilt_and_cloned(device, tmp_path):
    m = model(device, "fp32", seed=7)
    prompt = torch.randint(0, 50, (2, 6), generator=torch.Generator().manual_seed(3))
    want = m.generate(prompt, 5, temperature=0.0)
    path = str(tmp_path / "m.dlvk")
    m.save_weights(path)
    again = dl.load_model_file(path, device)
    assert torch.equal(again.generate(prompt, 5, temperature=0.0), want)
    assert model_from_architecture(m.architecture(), device).architecture() == m.architecture()
    c = m.clone().build()
    assert torch.equal(c.generate(prompt, 5, temperature=0.0), want)
    with pytest.raises(NotImplementedError):
        onnx.export_model(m, str(tmp_path / "m.onnx"), [2, 6])
