"""Loss functions (include/dlvk/loss/loss_functions.h:8-51,
src/loss/loss_functions.cpp).

`forward(pred, target)` / `backward(pred, target)` keep the reference
semantics on probabilities:
  CrossEntropyLoss       -sum t log(p + 1e-8) / B                    (:127-135)
  MeanSquaredError       mean((p - t)^2), grad 2 (p - t) / N           (:59-64)
  BinaryCrossEntropyLoss clamp eps 1e-7, mean, grad (p-t)/(p(1-p))/N   (:189-238)
CrossEntropyLoss.backward returns -t / (p + 1e-8) / B, the gradient w.r.t.
the softmax output, which the standard softmax Jacobian turns into the
(p - t) / B logits gradient the reference obtained with an identity softmax
backward.  Training uses `value_and_grad(..., from_logits=True)`: one fused
softmax + cross-entropy kernel producing the loss and dlogits together.
Targets may be int class ids or one-hot / probability rows.
"""
from __future__ import annotations

import torch

from .ops import core as K
from .ops import functional as Fn


def _to_probs(target: torch.Tensor, cols: int) -> torch.Tensor:
    if target.is_floating_point():
        return target.float()
    t = torch.zeros(target.numel(), cols, dtype=torch.float32, device=target.device)
    t[torch.arange(target.numel(), device=target.device), target.reshape(-1).long()] = 1.0
    return t


def _unwrap(x):
    if isinstance(x, torch.Tensor):
        return x
    from .tensor import Tensor as FacadeTensor

    return x.data if isinstance(x, FacadeTensor) else x


class LossFunction:
    fuses_softmax = False

    def forward(self, predictions, targets):
        raise NotImplementedError

    def backward(self, predictions, targets):
        raise NotImplementedError

    def value_and_grad(self, out, target, from_logits: bool = False):
        raise NotImplementedError

    __call__ = lambda self, p, t: self.forward(p, t)  # noqa: E731


class CrossEntropyLoss(LossFunction):
    fuses_softmax = True

    def forward(self, predictions, targets):
        p = _unwrap(predictions).float()
        p2 = p.reshape(-1, p.shape[-1])
        t = _to_probs(_unwrap(targets).to(p.device), p2.shape[1]).reshape(p2.shape)
        return -(t * torch.log(p2 + 1e-8)).sum() / p2.shape[0]

    def backward(self, predictions, targets):
        p = _unwrap(predictions)
        p2 = p.reshape(-1, p.shape[-1]).float()
        t = _to_probs(_unwrap(targets).to(p.device), p2.shape[1]).reshape(p2.shape)
        return (-t / (p2 + 1e-8) / p2.shape[0]).to(p.dtype).reshape(p.shape)

    def value_and_grad(self, out, target, from_logits: bool = False):
        out = _unwrap(out)
        target = _unwrap(target)
        rows = out.numel() // out.shape[-1]
        if from_logits:
            tgt = target.to(out.device)
            if not tgt.is_floating_point():
                tgt = tgt.to(torch.int32)
            loss, dl = Fn.softmax_cross_entropy(out.reshape(rows, out.shape[-1]), tgt.reshape(rows, -1)
                                                if tgt.is_floating_point() else tgt.reshape(rows),
                                                1.0 / rows)
            return loss, dl.reshape(out.shape)
        return self.forward(out, target), self.backward(out, target)


class LinearCrossEntropyLoss(LossFunction):
    """Cross entropy of a model's last Dense layer and softmax taken together:
    the loss and the gradients of hidden @ weight + bias without an array of
    logits, which for a large vocabulary is the largest of the step.

    hidden [..., E], weight [E, V] (also the transpose of a [V, E] embedding
    table), bias [V] or None, target int32 / int64 [...].  Targets outside
    [0, V) and `ignore_index` do not count; the mean is over those that do
    (CrossEntropyLoss divides by all rows), and 0 when there are none.  Under
    data parallelism every rank's mean is over its own counted rows and the
    ranks' gradients are averaged: with unequal padding that is not the mean
    over all ranks' counted rows (reduction "sum" weighs them alike).

    What it keeps is a block of rows at a time: in bf16 2 bytes a logit, at
    most max(256 MB, 4096 bytes a word), in fp32 4 bytes and, with gradients,
    6 more, at most max(640 MB, 20 KB a word).

    `Sequential.train_step`, `TrainStep` and the trainers take it in the place
    of CrossEntropyLoss for a model that ends in a Dense layer without
    activation (and a Softmax or none)."""

    fuses_head = True

    def __init__(self, reduction: str = "mean", ignore_index=None):
        if reduction not in ("mean", "sum", "none"):
            raise ValueError(f"reduction is mean, sum or none, got {reduction!r}")
        self.reduction, self.ignore_index = reduction, ignore_index

    @staticmethod
    def _rows(hidden, target):
        hidden, target = _unwrap(hidden), _unwrap(target)
        if target.shape != hidden.shape[:-1]:
            raise ValueError(f"hidden {tuple(hidden.shape)} needs a target of {tuple(hidden.shape[:-1])}, "
                             f"got {tuple(target.shape)}")
        if hidden.dim() != 2:
            hidden, target = hidden.reshape(-1, hidden.shape[-1]), target.reshape(-1)
        return hidden, target

    def forward(self, hidden, weight, target, bias=None, correct=None, counted=None):
        """The loss alone: a scalar, or with reduction "none" each row's (0 where it does not count).
        `counted` and `correct` (int64 device scalars) are increased by the rows that count and by
        those of them whose target has the largest logit."""
        x, t = self._rows(hidden, target)
        loss, rows, _, _, _ = K.linear_ce(x, _unwrap(weight), t, _unwrap(bias), self.ignore_index,
                                          self.reduction != "sum", False, correct=correct, counted=counted)
        return rows.reshape(_unwrap(target).shape) if self.reduction == "none" else loss

    def __call__(self, hidden, weight, target, bias=None):
        return self.forward(hidden, weight, target, bias)

    def value_and_grad(self, hidden, weight, target, bias=None, grad_scale=None):
        """(loss, dhidden, dweight, dbias): gradients of the loss (times the
        device scalar grad_scale) in the operands' layouts and types, dbias fp32."""
        if self.reduction == "none":
            raise ValueError("value_and_grad needs reduction mean or sum")
        x, t = self._rows(hidden, target)
        loss, _, dx, dw, db = K.linear_ce(x, _unwrap(weight), t, _unwrap(bias), self.ignore_index,
                                          self.reduction == "mean", True, grad_scale)
        return loss, dx.reshape(_unwrap(hidden).shape), dw, db

    def head_backward(self, head, hidden, target, grad_scale=None, correct=None, counted=None, loss_sum=None):
        """(loss, dhidden) for a Dense layer `head`, whose parameters receive
        their gradients (and whose grad-ready hooks fire).  `counted`, `correct`
        and `loss_sum` as in ops.core.linear_ce."""
        if self.reduction == "none":
            raise ValueError("training needs reduction mean or sum")
        x, t = self._rows(hidden, target)
        W, b = head.weight, head.bias
        loss, _, dx, _, _ = K.linear_ce(
            x, W.value, t, b.master if b is not None else None, self.ignore_index, self.reduction == "mean", True,
            grad_scale, dw_out=W.grad, dw_accumulate=W.take_accumulate_flag(), db_out=b.grad if b is not None else None,
            db_accumulate=b.take_accumulate_flag() if b is not None else False, correct=correct, counted=counted,
            loss_sum=loss_sum)
        W.grad_ready()
        if b is not None:
            b.grad_ready()
        return loss, dx.reshape(hidden.shape)


class MeanSquaredError(LossFunction):
    def forward(self, predictions, targets):
        p = _unwrap(predictions)
        loss, _ = K.pointwise_loss(p, _unwrap(targets).to(p.device), K.LOSS_MSE, 1.0 / p.numel(), 0.0, False)
        return loss

    def backward(self, predictions, targets):
        p = _unwrap(predictions)
        _, g = K.pointwise_loss(p, _unwrap(targets).to(p.device), K.LOSS_MSE, 1.0 / p.numel(), 1.0 / p.numel(), True)
        return g

    def value_and_grad(self, out, target, from_logits: bool = False):
        out = _unwrap(out)
        n = out.numel()
        return K.pointwise_loss(out, _unwrap(target).to(out.device), K.LOSS_MSE, 1.0 / n, 1.0 / n, True)


class BinaryCrossEntropyLoss(LossFunction):
    def forward(self, predictions, targets):
        p = _unwrap(predictions)
        loss, _ = K.pointwise_loss(p, _unwrap(targets).to(p.device), K.LOSS_BCE, 1.0 / p.numel(), 0.0, False)
        return loss

    def backward(self, predictions, targets):
        p = _unwrap(predictions)
        _, g = K.pointwise_loss(p, _unwrap(targets).to(p.device), K.LOSS_BCE, 1.0 / p.numel(), 1.0 / p.numel(), True)
        return g

    def value_and_grad(self, out, target, from_logits: bool = False):
        out = _unwrap(out)
        n = out.numel()
        return K.pointwise_loss(out, _unwrap(target).to(out.device), K.LOSS_BCE, 1.0 / n, 1.0 / n, True)


# Reference spellings.
MSELoss = MeanSquaredError
BCELoss = BinaryCrossEntropyLoss


class LossOpsGPU:
    """The reference's per-op loss entry points (include/dlvk/loss/loss_ops_gpu.h:10-60)
    over this library's loss kernels (softmax_loss.cu `pointwise_loss`;
    cross-entropy on probabilities as CrossEntropyLoss).  Each method returns
    its result tensor; the reference wrote it through an out-parameter and
    returned a success flag.  The semantics are the reference's CPU ones:

      mse_forward                    mean((p - t)^2)
      mse_backward                   2 (p - t) / N
      cross_entropy_forward          -sum t log(p + 1e-8) / B    (p: probabilities)
      cross_entropy_backward         -t / (p + 1e-8) / B
      binary_cross_entropy_forward   mean of -(t log p + (1 - t) log(1 - p)), p clamped to [eps, 1 - eps]
      binary_cross_entropy_backward  (p - t) / (p (1 - p)) / N with the same clamp

    The kernels clamp BCE probabilities at 1e-7; a larger `epsilon` clamps
    the predictions first, a smaller one is rejected."""

    def __init__(self, device=None):
        self.device = device

    def initialize(self) -> bool:
        return True

    def mse_forward(self, predictions, targets):
        return MeanSquaredError().forward(predictions, targets)

    def mse_backward(self, predictions, targets):
        return MeanSquaredError().backward(predictions, targets)

    def cross_entropy_forward(self, predictions, targets):
        return CrossEntropyLoss().forward(predictions, targets)

    def cross_entropy_backward(self, predictions, targets):
        return CrossEntropyLoss().backward(predictions, targets)

    @staticmethod
    def _clamped(predictions, epsilon: float):
        p = _unwrap(predictions)
        if epsilon < 1e-7:
            raise ValueError(f"epsilon {epsilon} is below the kernel's 1e-7 probability clamp")
        if epsilon > 1e-7:
            p = K.unary(p, K.UN_CLAMP, float(epsilon), 1.0 - float(epsilon))
        return p

    def binary_cross_entropy_forward(self, predictions, targets, epsilon: float = 1e-7):
        return BinaryCrossEntropyLoss().forward(self._clamped(predictions, epsilon), targets)

    def binary_cross_entropy_backward(self, predictions, targets, epsilon: float = 1e-7):
        return BinaryCrossEntropyLoss().backward(self._clamped(predictions, epsilon), targets)
