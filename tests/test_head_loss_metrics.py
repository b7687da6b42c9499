"""Loss and accuracy that training and evaluation report with a loss that takes
the head: means over the rows that count, however the data is cut into batches
and however unequal the padding is, for both reductions.
"""
import pytest
import torch

import dlvk_b200 as dl
from dlvk_b200.deployment.multi_gpu import MultiGPUTrainer
from dlvk_b200.models.sequential import Sequential
from test_linear_cross_entropy import exact

DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
V, E, N, S = 80, 64, 24, 10


def _data():
    g = torch.Generator().manual_seed(5)
    x = torch.randint(0, V, (N, S), generator=g, dtype=torch.int32)
    # from no padding in the first sequences to a single counted token in the last ones
    length = (S - torch.arange(N) * S // N).clamp(min=1)
    return x, torch.where(torch.arange(S)[None, :] < length[:, None], x, torch.full_like(x, -1))


def _model(device, right):
    """Token -> its embedding -> logits; `right`: the head is the embedding's transpose,
    so that a token's own word has by far the largest logit."""
    m = Sequential(device if device == "cpu" else "cuda:0", "fp32", seed=3)
    m.add_embedding(V, E, init_std=1.0)
    m.add_dense(E, V, use_bias=False, init_std=0.2)
    m.add_softmax()
    m.build()
    table, head = m.m_layers[0].weight, m.m_layers[1].weight
    if right:
        head.master.copy_(table.master.t())
        m.store.sync_value()
    return m, table.master.cpu().clone(), head.master.cpu().clone()


def _expected(x, y, table, head):
    """The mean over all counted rows and its limit (a few fp32 sums of batches' totals: 2^-20)."""
    value, lim = exact(table[x.reshape(-1).long()], head, y.reshape(-1), None)["loss"]
    return float(value), float(lim) + 2.0 ** -20 * float(value)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("right", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("batch", [5, 8, N])
def test_evaluation(device, right, reduction, batch):
    x, y = _data()
    m, table, head = _model(device, right)
    want, lim = _expected(x, y, table, head)
    loss = dl.LinearCrossEntropyLoss(reduction)
    batches = [(x[i:i + batch], y[i:i + batch]) for i in range(0, N, batch)]
    one = dl.ModelTrainer(m)
    one.compile(dl.SGD(0.0), loss)
    two = dl.Trainer(m, dl.SGD(0.0), loss)
    three = MultiGPUTrainer()
    three.initialize(m, dl.SGD(0.0), loss)
    results = [one.evaluate(x, y, batch), two.evaluate(batches, verbose=False), three.evaluate(batches)]
    for r in results:
        assert abs(r.loss - want) <= lim, (r.loss, want)
        if right:
            assert r.accuracy == 1.0
    hits = [r.accuracy * int((y >= 0).sum()) for r in results]
    assert all(abs(h - round(h)) < 1e-6 and h == hits[0] for h in hits)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("right", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("batch", [5, 8, N])
def test_training(device, right, reduction, batch):
    """SGD of rate 0: every step sees the same model."""
    x, y = _data()
    m, table, head = _model(device, right)
    want, lim = _expected(x, y, table, head)
    loss = dl.LinearCrossEntropyLoss(reduction)
    batches = [(x[i:i + batch], y[i:i + batch]) for i in range(0, N, batch)]
    one = dl.ModelTrainer(m)
    one.compile(dl.SGD(0.0), loss)
    two = dl.Trainer(m, dl.SGD(0.0), loss)
    three = MultiGPUTrainer()
    three.initialize(m, dl.SGD(0.0), loss)
    got = [one.fit(x, y, epochs=3, batch_size=batch, verbose=False, shuffle=False)[-1],
           two.fit(batches, epochs=3, verbose=False)[-1], three.train(batches, epochs=3)]
    for r in got:
        assert abs(r.loss - want) <= lim, (r.loss, want)
        if right:
            assert r.accuracy == 1.0


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_whose_rows_do_not_count(device):
    x, y = _data()
    m, _, _ = _model(device, True)
    step = dl.TrainStep(m, dl.LinearCrossEntropyLoss(), dl.SGD(0.0), metrics=True)
    for _ in range(4):
        step(x, torch.full_like(y, -1))
    assert step.epoch_metrics(reset=False) == (0.0, 0.0, 4 * N)
    step(x, y)
    loss, acc, samples = step.epoch_metrics()
    # the others' logits are tens below: exp of the difference is lost beside 1
    assert 0.0 <= loss <= 2.0 ** -20 and acc == 1.0 and samples == 5 * N
    assert step.epoch_totals() == (0.0, 0, 0.0, 0, 0)
    step.close()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("loss", [dl.LinearCrossEntropyLoss, dl.CrossEntropyLoss])
def test_a_training_step_in_evaluation_mode_is_refused(device, loss):
    """As with CrossEntropyLoss, whose output has no graph then: not a step of the head alone."""
    m, _, head = _model(device, False)
    x, y = _data()
    m.set_training(False)
    with pytest.raises(RuntimeError):
        m.train_step(x, y.clamp(min=0).to(m.dev.device), loss(), dl.SGD(0.1))
    with pytest.raises(RuntimeError):
        dl.TrainStep(m, loss(), dl.SGD(0.1), graph=False)(x, y.clamp(min=0))
    assert torch.equal(m.m_layers[1].weight.master.cpu(), head)
    m.set_training(True)
    m.train_step(x, y.clamp(min=0).to(m.dev.device), loss(), dl.SGD(0.1))
    assert not torch.equal(m.m_layers[1].weight.master.cpu(), head)
