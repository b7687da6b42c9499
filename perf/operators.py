"""Measured cases of the token-model operators: the cross entropy of a
vocabulary projection that keeps no logits, the embedding lookup with its
sorted gradient, and the global gradient norm with clipping.

`run` computes each operator either in its plain form (elementary torch
operations in 32 bits, 64 where 32 lose what matters) or, with `own` set,
through this package's public calls.  `exact` gives the values of the
operators' definitions in 64 bits.
"""
import math
import random

import torch

own = False

# The transformer configuration of the model zoo: 16 sequences of 512 tokens,
# width 1024, feed-forward 4096, 12 blocks, 32000 words.
_SEQ, _BATCH, _D, _FF, _BLOCKS, _VOCAB = 512, 16, 1024, 4096, 12, 32000

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # The training step of the zoo's transformer: its untied [width, words] head.
        {"name": "ce_train_config", "op": "ce", "rows": _BATCH * _SEQ, "width": _D, "words": _VOCAB, "dtype": "bf16",
         "tied": False, "bias": False, "grad": True},
        # The reduced model of a smoke run: launch latency counts.
        {"name": "ce_train_small", "op": "ce", "rows": 256, "width": 256, "words": 1024, "dtype": "bf16",
         "tied": False, "bias": False, "grad": True},
        # A head tied to the embedding table, an odd vocabulary and a ragged number of tokens.
        {"name": "ce_train_tied_ragged", "op": "ce", "rows": 1999, "width": 768, "words": 50257, "dtype": "bf16",
         "tied": True, "bias": False, "grad": True},
        # Perplexity of held-out text: each token's loss, no gradient.
        {"name": "ce_eval", "op": "ce", "rows": 4096, "width": _D, "words": _VOCAB, "dtype": "bf16",
         "tied": False, "bias": False, "grad": False},
        # A model kept in 32 bits, whose head has a bias.
        {"name": "ce_train_fp32_bias", "op": "ce", "rows": 768, "width": 512, "words": 10007, "dtype": "fp32",
         "tied": False, "bias": True, "grad": True},
        # The first layer of the zoo's transformer, scaled by the root of its width.
        {"name": "embed_lookup_config", "op": "lookup", "tokens": _BATCH * _SEQ, "width": _D, "words": _VOCAB,
         "dtype": "bf16", "pad": False},
        # One token for each of eight sequences being written.
        {"name": "embed_lookup_one_token", "op": "lookup", "tokens": 8, "width": _D, "words": _VOCAB, "dtype": "bf16",
         "pad": False},
        # Its gradient in the same step.
        {"name": "embed_grad_config", "op": "embed_grad", "tokens": _BATCH * _SEQ, "width": _D, "words": _VOCAB,
         "dtype": "bf16", "pad": False},
        # A padded batch of a small 32-bit model.
        {"name": "embed_grad_small_padded", "op": "embed_grad", "tokens": 1000, "width": 257, "words": 1024,
         "dtype": "fp32", "pad": True},
        # The norm of all gradients of the zoo's transformer, for a log line.
        {"name": "norm_config", "op": "norm", "layout": "transformer", "dtype": "fp32"},
        # The same gradients clipped into the optimizer's flat buffer.
        {"name": "clip_config", "op": "clip", "layout": "transformer", "dtype": "fp32"},
        # Many small tensors of both types at odd places: launches count.
        {"name": "clip_many_small", "op": "clip", "layout": "random", "tensors": 150, "largest": 20000, "shapes": 7,
         "dtype": "mixed"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "ce", "lookup", "embed_grad", "embed_grad", "norm", "clip"])
    if op == "ce":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        words = _log_uniform(rng, 500, 64000)
        width = 8 * _log_uniform(rng, 8, 192)
        if rng.random() < 0.2:
            width += rng.randint(1, 7)  # rows that no 16-byte step divides
        most = (_BATCH * _SEQ * _D * _VOCAB if dtype == "bf16" else 2 ** 33) // (width * words)
        rows = _log_uniform(rng, 1, max(1, min(16384, most)))
        return {"op": "ce", "rows": rows, "width": width, "words": words, "dtype": dtype,
                "tied": rng.random() < 0.5, "bias": rng.random() < 0.3, "grad": rng.random() < 0.75}
    if op in ("lookup", "embed_grad"):
        words = _log_uniform(rng, 100, 100000)
        width = _log_uniform(rng, 16, 2048)
        if rng.random() < 0.6:
            width = (width + 7) // 8 * 8
        words = max(100, min(words, _VOCAB * _D // width))
        return {"op": op, "tokens": _log_uniform(rng, 1, 16384), "width": width, "words": words,
                "dtype": rng.choice(["bf16", "bf16", "fp32"]), "pad": rng.random() < 0.4}
    return {"op": op, "layout": "random", "tensors": _log_uniform(rng, 1, 300), "largest": _log_uniform(rng, 10, 400000),
            "shapes": rng.randint(0, 10 ** 9), "dtype": rng.choice(["fp32", "bf16", "mixed"])}


def _tensors(case):
    """The gradients of a norm or clip case: [(shape, type, gap before it in its flat buffer)]."""
    if case["layout"] == "transformer":
        d, ff = _D, _FF
        block = [(d,), (d,), (d, 3 * d), (d, d), (d,), (d,), (d, ff), (ff,), (ff, d), (d,)]
        shapes = [(_VOCAB, d)] + block * _BLOCKS + [(d,), (d,), (d, _VOCAB)]
        return [(s, case["dtype"], 0) for s in shapes]
    rng = random.Random(case["shapes"])
    got = []
    for _ in range(case["tensors"]):
        n = _log_uniform(rng, 1, case["largest"])
        rows = rng.choice([1, 1, 2, 3, 16])
        shape = (n,) if rows == 1 or n < rows else (rows, n // rows)
        got.append((shape, rng.choice(["fp32", "bf16"]) if case["dtype"] == "mixed" else case["dtype"],
                    rng.choice([0, 0, 1, 3])))
    return got


# -------------------------------------------------------------------- the inputs
def _ids(count, words, g):
    """Token ids of text: the k-th commonest word comes about 1 / (k + 2.7) as often as the first."""
    weight = 1.0 / (torch.arange(words, device="cuda", dtype=torch.float64) + 2.7)
    upto = torch.cumsum(weight, 0)
    at = torch.rand(count, device="cuda", dtype=torch.float64, generator=g) * upto[-1]
    rank = torch.searchsorted(upto, at).clamp_(max=words - 1)
    return torch.randperm(words, device="cuda", generator=g)[rank]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "ce":
        n, d, v, t = case["rows"], case["width"], case["words"], _TYPES[case["dtype"]]
        target = _ids(n, v, g)
        # Logits of a model in training: they spread by about two, and a third
        # of the rows leans clearly to its word.
        w = torch.randn(v, d, device="cuda", generator=g) * (2.0 / math.sqrt(d))
        x = torch.randn(n, d, device="cuda", generator=g)
        lean = (torch.rand(n, 1, device="cuda", generator=g) < 0.33) * 3.0
        x += lean * w[target]
        s["x"] = x.to(t)
        s["w"] = w.to(t).t() if case["tied"] else w.t().contiguous().to(t)  # [width, words] either way
        s["bias"] = torch.randn(v, device="cuda", generator=g) if case["bias"] else None
        # a tenth of the tokens is not counted (padding, prompts)
        gone = torch.rand(n, device="cuda", generator=g) < 0.1
        gone[:1] = False
        s["target"] = torch.where(gone, torch.full_like(target, -1), target).to(torch.int32)
        return s
    if case["op"] in ("lookup", "embed_grad"):
        n, d, v, t = case["tokens"], case["width"], case["words"], _TYPES[case["dtype"]]
        ids = _ids(n, v, g).to(torch.int32)
        if case["pad"]:  # sequences end at odd places, and word 0 fills the rest
            ids = torch.where(torch.rand(n, device="cuda", generator=g) < 0.25, torch.zeros_like(ids), ids)
        s["ids"], s["scale"], s["padding"] = ids, math.sqrt(d), 0 if case["pad"] else None
        if case["op"] == "lookup":
            s["table"] = (torch.randn(v, d, device="cuda", generator=g) * 0.02).to(t)
        else:
            s["dy"] = (torch.randn(n, d, device="cuda", generator=g) * 1e-3).to(t)
        return s
    tensors = _tensors(case)
    room = {"fp32": 0, "bf16": 0}
    for shape, kind, gap in tensors:
        room[kind] += gap + math.prod(shape)
    source = {k: (torch.randn(room[k], device="cuda", generator=g) * 1e-3).to(_TYPES[k]) for k in room}
    at = {"fp32": 0, "bf16": 0}
    s["grads"] = []
    for shape, kind, gap in tensors:
        at[kind] += gap
        s["grads"].append(source[kind][at[kind]:at[kind] + math.prod(shape)].view(shape))
        at[kind] += math.prod(shape)
    s["max_norm"] = 1e-3
    if case["op"] == "clip":  # the optimizer's flat 32-bit buffer, one view for each gradient
        sizes = [math.prod(shape) for shape, _, _ in tensors]
        s["flat"] = torch.zeros(sum(sizes), device="cuda")
        s["out"] = [v.view(shape) for v, (shape, _, _) in zip(s["flat"].split(sizes), tensors)]
    return s


# ----------------------------------------------------------------- the operators
def _plain_ce(s):
    x, w, t = s["x"].float(), s["w"].float(), s["target"].long()
    counted = t >= 0
    at = t.clamp(min=0)[:, None]
    logits = x @ w
    if s["bias"] is not None:
        logits += s["bias"]
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    rows = (torch.log(total) + top - logits.gather(1, at))[:, 0]
    if not s["case"]["grad"]:
        return {"rows": rows * counted}
    share = counted.float() / counted.sum()
    loss = (rows * share).sum()
    dl = e / total
    dl.scatter_add_(1, at, torch.full_like(dl[:, :1], -1.0))
    dl *= share[:, None]
    got = {"loss": loss, "dx": (dl @ w.t()).to(s["x"].dtype), "dw": (x.t() @ dl).to(s["w"].dtype)}
    if s["bias"] is not None:
        got["dbias"] = dl.sum(0)
    return got


def _own_ce(s):
    from dlvk_b200 import LinearCrossEntropyLoss

    if not s["case"]["grad"]:
        return {"rows": LinearCrossEntropyLoss(reduction="none").forward(s["x"], s["w"], s["target"], s["bias"])}
    loss, dx, dw, dbias = LinearCrossEntropyLoss().value_and_grad(s["x"], s["w"], s["target"], s["bias"])
    got = {"loss": loss, "dx": dx, "dw": dw}
    if dbias is not None:
        got["dbias"] = dbias
    return got


def _plain_embed_grad(s):
    ids, dy = s["ids"].long(), s["dy"].float() * s["scale"]
    if s["padding"] is not None:
        dy = dy * (ids != s["padding"])[:, None]
    return torch.zeros(s["case"]["words"], dy.shape[1], device=dy.device).index_add_(0, ids, dy)


def _plain_norm(grads):
    flat = torch.cat([t.reshape(-1).float() for t in grads])
    return flat, torch.sqrt((flat.double() * flat.double()).sum())


def run(s):
    op = s["case"]["op"]
    if own:
        from dlvk_b200 import GradientClipping
        from dlvk_b200.ops import nn

        if op == "ce":
            return _own_ce(s)
        if op == "lookup":
            return nn.embedding_lookup(s["ids"], s["table"], scale=s["scale"])
        if op == "embed_grad":
            return nn.embedding_grad(s["ids"], s["dy"], s["case"]["words"], scale=s["scale"], padding_idx=s["padding"])
        if op == "norm":
            return GradientClipping.global_norm(s["grads"])
        return {"norm": GradientClipping.clip_global_norm(s["grads"], s["max_norm"], out=s["out"]), "out": s["flat"]}
    if op == "ce":
        return _plain_ce(s)
    if op == "lookup":
        return (s["table"][s["ids"].long()].float() * s["scale"]).to(s["table"].dtype)
    if op == "embed_grad":
        return _plain_embed_grad(s)
    flat, norm = _plain_norm(s["grads"])
    if op == "norm":
        return norm.float()
    share = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    s["flat"].copy_(flat * share.float())
    return {"norm": norm.float(), "out": s["flat"]}


# ------------------------------------------------------------------------ the work
def work(case):
    if case["op"] == "ce":
        n, d, v = case["rows"], case["width"], case["words"]
        size = _TYPES[case["dtype"]].itemsize
        read = size * (n * d + d * v) + 4 * n + (4 * v if case["bias"] else 0)
        wrote = size * (n * d + d * v) + (4 * v if case["bias"] else 0) + 4 if case["grad"] else 4 * n
        return {"bytes": read + wrote, "flops": (6 if case["grad"] else 2) * n * d * v}
    if case["op"] in ("lookup", "embed_grad"):
        n, d, v = case["tokens"], case["width"], case["words"]
        size = _TYPES[case["dtype"]].itemsize
        if case["op"] == "lookup":
            return {"bytes": 4 * n + 2 * size * n * d, "flops": n * d}
        return {"bytes": 4 * n + size * n * d + 4 * v * d, "flops": n * d}
    sizes = [(math.prod(shape), _TYPES[kind].itemsize) for shape, kind, _ in _tensors(case)]
    read = sum(n * size for n, size in sizes)
    count = sum(n for n, _ in sizes)
    if case["op"] == "norm":
        return {"bytes": read + 4, "flops": 2 * count}
    return {"bytes": read + 4 * count + 4, "flops": 3 * count}


# --------------------------------------------------------------- values in 64 bits
def _exact_ce(s):
    x, w, target = s["x"].double(), s["w"].double(), s["target"].long()
    bias = s["bias"].double() if s["bias"] is not None else None
    n, v = x.shape[0], w.shape[1]
    count = int((target >= 0).sum())
    rows = torch.zeros(n, dtype=torch.float64, device=x.device)
    dx = torch.zeros_like(x)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    dbias = torch.zeros(v, dtype=torch.float64, device=x.device)
    for a in range(0, n, 1024):
        t = target[a:a + 1024]
        keep = torch.nonzero(t >= 0)[:, 0]
        z = x[a:a + 1024][keep] @ w
        if bias is not None:
            z = z + bias
        lse = torch.logsumexp(z, 1)
        here = torch.arange(keep.numel(), device=x.device)
        rows[a + keep] = lse - z[here, t[keep]]
        if not s["case"]["grad"]:
            continue
        p = torch.exp(z - lse[:, None])
        p[here, t[keep]] -= 1.0
        p /= count
        dx[a + keep] = p @ w.t()
        dw += x[a:a + 1024][keep].t() @ p
        dbias += p.sum(0)
    if not s["case"]["grad"]:
        return {"rows": rows}
    got = {"loss": rows.sum() / count, "dx": dx, "dw": dw}
    if bias is not None:
        got["dbias"] = dbias
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ce":
        return _exact_ce(s)
    if case["op"] == "lookup":
        return torch.index_select(s["table"].double(), 0, s["ids"].long()) * s["scale"]
    if case["op"] == "embed_grad":
        # differences of running sums over the tokens in the order of their words
        ids = s["ids"].long()
        keep = ids >= 0 if s["padding"] is None else ids != s["padding"]
        order, at = torch.sort(ids[keep])
        upto = torch.cumsum(s["dy"][keep][at].double(), 0)
        upto = torch.cat([torch.zeros_like(upto[:1]) if at.numel() else upto.new_zeros(1, s["dy"].shape[1]), upto])
        word = torch.arange(case["words"], device=ids.device)
        return (upto[torch.searchsorted(order, word, right=True)] - upto[torch.searchsorted(order, word)]) * s["scale"]
    total = sum(float(t.double().square().sum()) for t in s["grads"])
    norm = torch.tensor(math.sqrt(total), dtype=torch.float64)
    if case["op"] == "norm":
        return norm
    share = min(1.0, s["max_norm"] / (math.sqrt(total) + 1e-6))
    return {"norm": norm, "out": torch.cat([t.double().reshape(-1) * share for t in s["grads"]])}
