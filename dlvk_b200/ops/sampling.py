"""The choice of the next word from its logits.  GPU tensors run
csrc/kernels/sampling.cu, CPU tensors the same rule in torch."""
from __future__ import annotations

import math

import torch

from .core import N, native

MOST_WORDS = 1 << 18
_ONE = 2.0 ** 44  # weights are summed as whole numbers, in steps of 2^-44 of the largest


def _setting(name, v, kind, rows, device):
    """(one value, or a default, and a tensor of one for each row, or None)."""
    if not torch.is_tensor(v):
        return v, None
    if v.dtype != kind or tuple(v.shape) != (rows,):
        raise ValueError(f"{name}: one value, or a {kind} tensor [{rows}]; got {v.dtype} {tuple(v.shape)}")
    if v.device != device:
        raise ValueError(f"{name} is on {v.device}, the logits on {device}")
    return 0, v


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """The next word of every row, int32 [...], from logits [..., words] (fp32
    or bf16, at most 2^18 words) and uniform numbers of [0, 1) (fp32 [...]).

    Words are taken in descending order of their logits, equal ones in that of
    their numbers: the first `top_k`; of these the fewest whose share of their
    weights' sum reaches `top_p`; of these the ones at least `min_p` times as
    likely as the first.  weight = exp((logit - largest) / temperature).  The
    answer is, in the order of the numbers, the first word left whose running
    sum of weights passes uniform times their total.

    Each setting is one value, or a tensor of one for each row (int32 for
    top_k, fp32 otherwise).  temperature <= 0 takes the likeliest word; top_k
    <= 0, top_p >= 1 and min_p <= 0 cut nothing.  A NaN logit counts as
    -infinity, and a setting that is NaN as the one that cuts nothing
    (temperature: as 0).  A row of nothing but -infinity gives -1.  Sums are
    exact in steps of 2^-44 of the largest weight, so the answer does not
    depend on how they are made.
    """
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits are fp32 or bf16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MOST_WORDS:
        raise ValueError(f"logits are [..., 1 to {MOST_WORDS} words], got {tuple(logits.shape)}")
    shape, words = logits.shape[:-1], logits.shape[-1]
    if uniform.dtype != torch.float32 or uniform.shape != shape:
        raise ValueError(f"uniform numbers are fp32 {tuple(shape)}, got {uniform.dtype} {tuple(uniform.shape)}")
    if uniform.device != logits.device:
        raise ValueError(f"uniform numbers on {uniform.device}, logits on {logits.device}")
    rows = math.prod(shape)
    x = logits if logits.dim() == 2 else logits.reshape(rows, words)
    given = [_setting(name, v, kind, rows, logits.device) for name, v, kind in
             (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
              ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32))]
    (t, ts), (k, ks), (p, ps), (m, ms) = given
    if native(logits):
        return N().sample_tokens(x, uniform.reshape(rows), float(t), int(k), float(p), float(m), ts, ks, ps,
                                 ms).reshape(shape)
    col = lambda v, vs, kind: (vs.to(kind) if vs is not None else torch.full((rows,), v, dtype=kind))[:, None]  # noqa: E731
    t, p, m = (col(v, vs, torch.float64) for v, vs in (given[0], given[2], given[3]))
    k = col(int(k), ks, torch.int64)
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    if not rows:
        return torch.zeros(shape, dtype=torch.int32)
    top = x.amax(1, keepdim=True)
    greedy = ~(t > 0)
    weight = torch.exp((x - top) / torch.where(greedy, 1.0, t))
    weight = torch.where(x == top, 1.0, torch.where(torch.isfinite(weight) & (x > -math.inf), weight, 0.0))
    weight = torch.round(weight * _ONE).long()
    falling, order = torch.sort(x, dim=1, descending=True, stable=True)
    place = torch.arange(words)[None]
    sw = torch.gather(weight, 1, order) * ((k <= 0) | (place < k))
    upto = torch.cumsum(sw, 1)
    want = torch.ceil(p.clamp(0, 1).nan_to_num(1.0) * upto[:, -1:].double()).long().clamp(min=1)
    keep = ~(p < 1) | (upto - sw < want)
    least = torch.ceil(m.clamp(0, 1).nan_to_num(0.0) * _ONE).long()
    keep &= (~(m > 0) | (sw >= least)) & (~greedy | (place < 1))
    weight = torch.zeros_like(weight).scatter_(1, order, sw * keep)
    upto = torch.cumsum(weight, 1)
    u = uniform.reshape(rows, 1).double().nan_to_num(0.0).clamp(min=0)
    want = torch.minimum((u.clamp(max=1) * upto[:, -1:].double()).long(), upto[:, -1:] - 1)
    token = (upto > want).to(torch.uint8).argmax(1)
    return torch.where(falling[:, 0] > -math.inf, token, -1).to(torch.int32).reshape(shape)
