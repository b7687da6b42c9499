"""StateSpaceLayer and Sequential.generate in the cases at their borders: models
that end in the layer itself."""
import pytest
import torch

import dlvk_b200 as dl
from dlvk_b200.models.sequential import Sequential
from test_state_space_layer import layer_ref

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
WORDS = 40


def ending_in(what, device):
    """A model whose last layer, before a Softmax or none, is `what`."""
    m = Sequential(device, "fp32", seed=5)
    m.add_embedding(WORDS, WORDS)
    if what == "state space":
        m.add_state_space(WORDS, residual=True)
    elif what == "state space, softmax":
        m.add_state_space(WORDS, residual=True).add_softmax()
    elif what == "residual":
        m.add_dense(WORDS, WORDS).add(dl.ResidualLayer(dl.StateSpaceLayer(WORDS, d_state=5)))
    elif what == "two, dense":
        m.add_state_space(WORDS, residual=True).add_state_space(WORDS, residual=True).add_dense(WORDS, WORDS)
    elif what == "embedding, softmax":
        m.add_softmax()
    return m.build()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("what", ["state space", "state space, softmax", "residual", "two, dense", "embedding",
                                  "embedding, softmax"])
def test_generate_takes_the_last_token_that_counts(device, what):
    """Every word of a padded batch is the likeliest after its sequence's own
    tokens, by the whole model's logits of them.  The two ways make the same fp32
    sums of at most 80 terms in other orders (3 2^-17 each on the GPU's split
    products), three layers deep: a word may be another one of the likeliest
    within 2^-8 of the largest logit."""
    m = ending_in(what, device)
    g = torch.Generator().manual_seed(3)
    n = [7, 2, 1, 5]
    prompt = torch.randint(0, WORDS, (4, 7), generator=g, dtype=torch.int32)
    for i, k in enumerate(n):
        prompt[i, k:] = (prompt[i, k - 1] + 1) % WORDS  # not the last word that counts
    got = m.generate(prompt, 4, lengths=n, temperature=0.0)
    m.set_training(False)
    for i, k in enumerate(n):
        seq = prompt[i, :k].tolist()
        for word in got[i].tolist():
            z = m.forward_logits(torch.tensor([seq], dtype=torch.int32)).detach()[0, -1].float().cpu()
            assert float(z.max() - z[word]) <= 2.0 ** -8 * float(z.abs().max()), (i, seq, word, int(z.argmax()))
            seq.append(word)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,T", [(0, 5), (2, 0), (0, 0)])
@pytest.mark.parametrize("groups", [1, 2])
def test_layer_of_no_sequences_or_tokens(device, B, T, groups):
    dl.manual_seed(3)
    layer = dl.StateSpaceLayer(16, groups=groups, residual=True)
    layer.to(device, torch.float32)
    x = torch.zeros(B, T, 16, device=device)
    y = layer.forward(x)
    assert y.shape == (B, T, 16)
    assert layer.backward(torch.zeros_like(y)).shape == (B, T, 16)
    assert all(not p.grad.any() for p in layer.parameters())
    start = layer.init_state(B)
    start.conv.normal_()
    start.scan.normal_()
    y, state = layer.prompt(x, start)
    assert y.shape == (B, T, 16) and torch.equal(state.conv, start.conv) and torch.equal(state.scan, start.scan)
    if B == 0:
        assert layer.step(x.new_zeros(0, 16), state).shape == (0, 16)


@pytest.mark.parametrize("device", DEVICES)
def test_states_are_kept_for_a_backward_pass_alone(device, monkeypatch):
    """Where no gradient is wanted the scan keeps no states between spans; outputs
    are the same bits."""
    from dlvk_b200.ops import ssm

    kept = []
    scan = ssm.state_scan_fwd

    def seen(*args, save=False, **kw):
        got = scan(*args, save=save, **kw)
        kept.append(got[2] is not None)
        return got

    monkeypatch.setattr(ssm, "state_scan_fwd", seen)
    m = Sequential(device, "fp32", seed=2)
    m.add_embedding(WORDS, 16).add_state_space(16, residual=True).add_dense(16, WORDS).build()
    x = torch.randint(0, WORDS, (2, 37), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(device)
    trained = m.forward(x)
    m.set_training(False)
    assert torch.equal(m.forward(x), trained)
    assert kept == [True, False]
    with torch.no_grad():
        layer = dl.StateSpaceLayer(16)
        layer.to(device, torch.float32)
        layer.track = False
        layer.forward(torch.zeros(2, 5, 16, device=device))
    assert kept == [True, False, False]
    layer.track = True
    layer.forward(torch.zeros(2, 5, 16, device=device))
    assert layer.backward(torch.ones(2, 5, 16, device=device)).shape == (2, 5, 16) and kept[-1]


@pytest.mark.gpu
@pytest.mark.parametrize("d_model,groups,kw", [(100, 1, {}), (100, 4, {}), (33, 1, dict(d_state=5, d_conv=3)),
                                               (72, 3, dict(dt_rank=9, d_state=33))])
def test_bf16_layer_of_odd_columns(d_model, groups, kw):
    """Columns of dt, b and c that begin at no multiple of four elements.  As in
    test_state_space_layer: eight roundings of 2^-8 in a row to the output, 24 with
    the way back, of values whose sums grow errors no more than themselves."""
    dl.manual_seed(3)
    layer = dl.StateSpaceLayer(d_model, groups=groups, residual=True, **kw)
    layer.to("cuda", torch.bfloat16)
    g = torch.Generator().manual_seed(6)
    x, dy = (torch.randn(2, 70, d_model, generator=g).bfloat16() for _ in range(2))
    y = layer.forward(x.cuda())
    dx = layer.backward(dy.cuda())
    xr = x.double().requires_grad_(True)
    ref, p = layer_ref(layer, xr)
    names = list(p)
    grads = torch.autograd.grad(ref, [xr] + [p[k] for k in names], dy.double())
    off = lambda a, b: float((a.detach().cpu().double() - b).norm() / b.norm())  # noqa: E731
    assert off(y, ref) <= 8 * 2.0 ** -8 and off(dx, grads[0]) <= 24 * 2.0 ** -8
    for k, r in zip(names, grads[1:]):
        assert off(getattr(layer, k).grad, r) <= 24 * 2.0 ** -8, k
