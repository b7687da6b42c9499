"""Measured cases of the operators of a token model with states: the short
causal convolution and the selective state space scan (training, prompts and
single tokens), and the choice of the next word from its logits.

`run` computes each operator either in its plain form (elementary torch
operations in 32 bits, 64 where 32 lose what matters) or, with `own` set,
through this package's public calls.  `exact` gives the values of the
operators' definitions in 64 bits.
"""
import math

import torch

own = False

# The transformer configuration of the model zoo has 16 sequences of 512
# tokens, width 1024, 32000 words; a state space layer of that width works on
# twice the width, with 16 states a channel, a convolution over 4 tokens and
# steps from a projection of 1024 / 16 = 64 columns.
_BATCH, _SEQ, _INNER, _STATES, _TAPS, _RANK, _VOCAB = 16, 512, 2048, 16, 4, 64, 32000

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------- the cases
def _scan(name, op, batch, tokens, channels, states, groups, dtype, gate=True, state=False, ragged=False):
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "channels": channels, "states": states,
            "groups": groups, "dtype": dtype, "gate": gate, "state": state, "ragged": ragged}


def _conv(name, op, batch, tokens, channels, taps, dtype, bias=True, silu=True, state=False, ragged=False):
    return {"name": name, "op": op, "batch": batch, "tokens": tokens, "channels": channels, "taps": taps,
            "dtype": dtype, "bias": bias, "silu": silu, "state": state, "ragged": ragged}


def _sample(name, rows, words, dtype, temperature, top_k, top_p, min_p, masked=0.0, per_row=False):
    return {"name": name, "op": "sample", "rows": rows, "words": words, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "masked": masked, "per_row": per_row}


def listed():
    return [
        # The training step of a layer at the zoo's transformer configuration, forward and backward.
        _scan("scan_train_config", "scan_train", _BATCH, _SEQ, _INNER, _STATES, 1, "bf16"),
        # A small model in 32 bits on a padded batch of odd lengths.
        _scan("scan_train_small", "scan_train", 3, 77, 200, 5, 1, "fp32", ragged=True),
        # One long document read in, its state kept for what follows.
        _scan("scan_prompt_long", "scan_prompt", 1, 16384, _INNER, _STATES, 1, "bf16"),
        # Eight conversations of different lengths that go on from their states.
        _scan("scan_prompt_ragged", "scan_prompt", 8, 700, _INNER, _STATES, 1, "bf16", state=True, ragged=True),
        # A token each for 64 sequences being written.
        _scan("scan_step_batch", "scan_step", 64, 1, _INNER, _STATES, 1, "bf16"),
        # A token of a single sequence: launch latency counts.
        _scan("scan_step_one", "scan_step", 1, 1, _INNER, _STATES, 1, "bf16"),
        # The convolution of the same training step, forward and backward.
        _conv("conv_train_config", "conv_train", _BATCH, _SEQ, _INNER, _TAPS, "bf16"),
        # Prompts of odd lengths and width in 32 bits that go on from earlier tokens.
        _conv("conv_prompt_ragged", "conv_prompt", 5, 1037, 1001, _TAPS, "fp32", state=True, ragged=True),
        # A token each for 64 sequences.
        _conv("conv_step_batch", "conv_step", 64, 1, _INNER, _TAPS, "bf16"),
        # The next words of 64 sequences with the usual settings of a chat.
        _sample("sample_batch", 64, _VOCAB, "bf16", 0.8, 50, 0.95, 0.0),
        # The next word of one sequence over an odd vocabulary, from the nucleus alone.
        _sample("sample_one", 1, 50257, "fp32", 0.7, 0, 0.9, 0.0),
        # A large batch over a large vocabulary, each row with settings of its own, some words masked.
        _sample("sample_large", 256, 128000, "fp32", 1.0, 0, 1.0, 0.0, masked=0.3, per_row=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, hi):
    n = _log_uniform(rng, 16, hi)
    return (n + 7) // 8 * 8 if rng.random() < 0.7 else n


def draw(rng):
    op = rng.choice(["scan_train", "scan_train", "scan_prompt", "scan_prompt", "scan_step", "conv_train",
                     "conv_prompt", "conv_step", "sample", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "sample":
        words = _log_uniform(rng, 100, 128000)
        return {"op": op, "rows": _log_uniform(rng, 1, 256), "words": words, "dtype": dtype,
                "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]),
                "top_k": rng.choice([0, 0, 1, 20, 50, 200, 5000]), "top_p": rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]),
                "min_p": rng.choice([0.0, 0.0, 0.0, 0.02, 0.1]), "masked": rng.choice([0.0, 0.0, 0.3, 0.95]),
                "per_row": rng.random() < 0.3}
    channels = _channels(rng, 4096)
    if op.startswith("conv"):
        got = {"op": op, "channels": channels, "taps": rng.choice([2, 3, 4, 4, 4, 4]), "dtype": dtype,
               "bias": rng.random() < 0.8, "silu": rng.random() < 0.8}
        room = _BATCH * _SEQ * _INNER // channels
    else:
        states = rng.choice([16, 16, 16, 64, rng.randint(1, 64)])
        groups = rng.choice([1, 1, 1, 2, 4])
        channels = (channels + groups - 1) // groups * groups
        got = {"op": op, "channels": channels, "states": states, "groups": groups, "dtype": dtype,
               "gate": rng.random() < 0.8}
        room = (2 if op == "scan_prompt" else 1) * _BATCH * _SEQ * _INNER * _STATES // (channels * states)
    if op.endswith("step"):
        got.update(batch=_log_uniform(rng, 1, min(512, room)), tokens=1, state=True, ragged=False)
        return got
    tokens = _log_uniform(rng, 1, min(16384 if op.endswith("prompt") else 4096, room))
    batch = _log_uniform(rng, 1, max(1, min(64, room // tokens)))
    got.update(batch=batch, tokens=tokens, state=op.endswith("prompt") and rng.random() < 0.5,
               ragged=rng.random() < 0.4)
    return got


# -------------------------------------------------------------------- the inputs
def _lengths(case, g):
    """Lengths of a padded batch: one sequence fills it, another may be empty."""
    if not case["ragged"]:
        return None
    n = torch.randint(0, case["tokens"] + 1, (case["batch"],), device="cuda", generator=g)
    n[0] = case["tokens"]
    return n.to(torch.int32)


def _prepare_conv(case, g):
    b, t, d, k, dt = case["batch"], case["tokens"], case["channels"], case["taps"], _TYPES[case["dtype"]]
    # x is the first half of a projection's columns, whose second half is the gate
    s = {"x": torch.randn(b, t, 2 * d, device="cuda", generator=g).to(dt)[:, :, :d], "lengths": _lengths(case, g)}
    s["weight"] = (torch.rand(d, k, device="cuda", generator=g) * 2 - 1) / math.sqrt(k)
    s["bias"] = (torch.rand(d, device="cuda", generator=g) * 2 - 1) / math.sqrt(k) if case["bias"] else None
    s["state"] = None
    if case["state"] or case["op"] == "conv_step":
        s["state"] = torch.randn(b, k - 1, d, device="cuda", generator=g).to(dt)
    if case["op"] == "conv_step":
        s["x"] = s["x"][:, 0]
        s["next"] = torch.empty_like(s["state"])
    if case["op"] == "conv_train":
        s["dy"] = (torch.randn(b, t, d, device="cuda", generator=g) * 1e-2).to(dt)
    return s


def _prepare_scan(case, g):
    b, t, d, n, dt = case["batch"], case["tokens"], case["channels"], case["states"], _TYPES[case["dtype"]]
    gn = case["groups"] * n
    randn = lambda *size: torch.randn(*size, device="cuda", generator=g)  # noqa: E731
    u = randn(b, t, d)
    s = {"u": (u * torch.sigmoid(u)).to(dt), "lengths": _lengths(case, g)}
    # the steps' projection before its bias; b and c follow the low-rank columns in one product's output
    s["dt"] = (randn(b, t, d) * 0.5).to(dt)
    dbc = randn(b, t, _RANK + 2 * gn).to(dt)
    s["b"] = dbc[:, :, _RANK:_RANK + gn].unflatten(2, (case["groups"], n))
    s["c"] = dbc[:, :, _RANK + gn:].unflatten(2, (case["groups"], n))
    s["z"] = randn(b, t, 2 * d).to(dt)[:, :, d:] if case["gate"] else None
    # decays of 1 to n a unit of time, steps of 0.001 to 0.1 units
    s["a_log"] = torch.log(torch.arange(1, n + 1, device="cuda", dtype=torch.float32)).repeat(d, 1) + 0.1 * randn(d, n)
    s["skip"] = 1.0 + 0.1 * randn(d)
    step = torch.exp(torch.rand(d, device="cuda", generator=g) * math.log(100.0) + math.log(1e-3))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus of it is the step
    s["state"] = randn(b, d, n) if case["state"] or case["op"] == "scan_step" else None
    if case["op"] == "scan_step":
        for k in ("u", "dt", "b", "c", "z"):
            s[k] = s[k][:, 0] if s[k] is not None else None
        s["next"] = torch.empty_like(s["state"])
    if case["op"] == "scan_train":
        s["dy"] = (randn(b, t, d) * 1e-2).to(dt)
    return s


def _prepare_sample(case, g):
    r, v, dt = case["rows"], case["words"], _TYPES[case["dtype"]]
    # Logits of a language model: words differ in how common they are, and
    # each row leans to some tens of its own.
    common = -torch.log(torch.arange(v, device="cuda", dtype=torch.float32) + 2.7)
    x = common[torch.randperm(v, device="cuda", generator=g)] + 1.5 * torch.randn(r, v, device="cuda", generator=g)
    lean = torch.randint(0, v, (r, min(v, 30)), device="cuda", generator=g)
    x.scatter_add_(1, lean, 6.0 + 2.0 * torch.randn(lean.shape, device="cuda", generator=g))
    if case["masked"]:  # words that a grammar does not allow, by either of the usual masks
        gone = torch.rand(r, v, device="cuda", generator=g) < case["masked"]
        low = torch.where(torch.arange(r, device="cuda") % 2 == 0, -math.inf, torch.finfo(dt).min)[:, None]
        x = torch.where(gone, low, x)
        if r > 2:
            x[r // 2] = -math.inf  # a row without any word
    s = {"logits": x.to(dt), "uniform": torch.rand(r, device="cuda", generator=g)}
    s["set"] = {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    if case["per_row"]:
        pick = lambda values, kind: torch.tensor(values, dtype=kind, device="cuda")[  # noqa: E731
            torch.randint(0, len(values), (r,), device="cuda", generator=g)]
        s["set"] = {"temperature": pick([0.0, 0.5, 0.7, 1.0, 1.3], torch.float32),
                    "top_k": pick([0, 0, 1, 40, 1000], torch.int32),
                    "top_p": pick([0.5, 0.9, 0.95, 1.0], torch.float32),
                    "min_p": pick([0.0, 0.0, 0.05], torch.float32)}
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["op"].split("_")[0]
    s = {"conv": _prepare_conv, "scan": _prepare_scan, "sample": _prepare_sample}[kind](case, g)
    s["case"] = case
    return s


# --------------------------------------------------------- the operators, plain
def _counts(s, tokens):
    """[batch, tokens, 1]: which positions a sequence has."""
    return (torch.arange(tokens, device="cuda")[None, :] < s["lengths"][:, None].long())[..., None]


def _silu(x):
    return x * torch.sigmoid(x)


def _silu_slope(x):
    p = torch.sigmoid(x)
    return p * (1 + x * (1 - p))


def _conv_windows(s):
    """The tokens with the ones before them, in 32 bits, and each position's window of taps (a view)."""
    x, k = s["x"].float(), s["weight"].shape[1]
    x = x[:, None] if x.dim() == 2 else x
    before = s["state"].float() if s["state"] is not None else x.new_zeros(x.shape[0], k - 1, x.shape[2])
    if s["lengths"] is not None:
        x = torch.where(_counts(s, x.shape[1]), x, torch.zeros_like(x))
    x = torch.cat([before, x], 1)
    return x, x.unfold(1, k, 1)  # [batch, tokens, channels, taps]


def _plain_conv(s):
    case, k = s["case"], s["weight"].shape[1]
    x, windows = _conv_windows(s)
    tokens = x.shape[1] - (k - 1)
    pre = (windows * s["weight"]).sum(3)
    if s["bias"] is not None:
        pre = pre + s["bias"]
    y = _silu(pre) if case["silu"] else pre
    if s["lengths"] is not None:
        y = y * _counts(s, tokens)
    y = y.to(s["x"].dtype)
    if case["op"] == "conv_train":
        g = s["dy"].float()
        if s["lengths"] is not None:
            g = torch.where(_counts(s, tokens), g, torch.zeros_like(g))
        if case["silu"]:
            g = g * _silu_slope(pre)
        # dx[t] = sum over taps j of w[j] g[t + k - 1 - j]
        after = torch.cat([g, g.new_zeros(g.shape[0], k - 1, g.shape[2])], 1).unfold(1, k, 1)
        got = {"y": y, "dx": (after * s["weight"].flip(1)).sum(3).to(y.dtype),
               "dweight": (windows * g[..., None]).sum((0, 1), dtype=torch.float64).float()}
        if s["bias"] is not None:
            got["dbias"] = g.sum((0, 1), dtype=torch.float64).float()
        return got
    if case["op"] == "conv_step":
        s["next"].copy_(x[:, 1:])
        return {"y": y[:, 0], "state": s["next"]}
    # the last k - 1 tokens that count
    end = s["lengths"].long() if s["lengths"] is not None else torch.full((x.shape[0],), tokens, device="cuda")
    at = end[:, None] + torch.arange(k - 1, device="cuda")
    return {"y": y, "state": torch.gather(x, 1, at[..., None].expand(-1, -1, x.shape[2])).to(s["x"].dtype)}


def _running(decay, x):
    """h[t] = decay[t] h[t-1] + x[t] along dimension 1, by doubling spans; both arguments are used up."""
    step = 1
    while step < x.shape[1]:
        x[:, step:] += decay[:, step:] * x[:, :-step]
        decay[:, step:] = decay[:, step:] * decay[:, :-step]
        step *= 2
    return x


def _scan_parts(s):
    """(tokens' inputs and steps [batch, tokens, channels], b and c [batch, tokens, groups, 1, states], a [channels, states])."""
    one = s["u"].dim() == 2
    grow = lambda v: v[:, None].float() if one else v.float()  # noqa: E731
    u, raw = grow(s["u"]), grow(s["dt"]) + s["dt_bias"]
    step = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    if s["lengths"] is not None:  # a step of no time changes no state
        step = step * _counts(s, step.shape[1])
    return u, raw, step, grow(s["b"])[:, :, :, None], grow(s["c"])[:, :, :, None], -torch.exp(s["a_log"])


def _plain_scan(s):
    case = s["case"]
    u, raw, step, b, c, a = _scan_parts(s)
    groups = case["groups"]
    split = lambda v: v.unflatten(2, (groups, -1))  # [batch, tokens, groups, channels of one, ...]  # noqa: E731
    decay = torch.exp(split(step[..., None] * a))
    h = split(step * u)[..., None] * b
    if s["state"] is not None:
        h[:, 0] += decay[:, 0] * s["state"].unflatten(1, (groups, -1))
    keep = decay.clone() if case["op"] == "scan_train" else None
    h = _running(decay, h)
    pre = (h * c).sum(4).flatten(2) + s["skip"] * u
    z = s["z"] if s["z"] is None or s["z"].dim() == 3 else s["z"][:, None]
    y = pre * _silu(z.float()) if z is not None else pre
    if s["lengths"] is not None:
        y = torch.where(_counts(s, y.shape[1]), y, torch.zeros_like(y))
    y = y.to(s["u"].dtype)
    if case["op"] == "scan_prompt":
        return {"y": y, "state": h[:, -1].flatten(1, 2).contiguous()}
    if case["op"] == "scan_step":
        s["next"].copy_(h[:, -1].flatten(1, 2))
        return {"y": y[:, 0], "state": s["next"]}
    # gradients
    dy = s["dy"].float()
    if s["lengths"] is not None:
        dy = torch.where(_counts(s, dy.shape[1]), dy, torch.zeros_like(dy))
    got = {"y": y}
    if z is not None:
        got["dz"] = (dy * pre * _silu_slope(z.float())).to(y.dtype)
        dy = dy * _silu(z.float())
    # g[t] = c[t] dy[t] + decay[t + 1] g[t + 1]
    g = split(dy)[..., None] * c
    got["dc"] = (h * split(dy)[..., None]).sum(3).to(y.dtype)
    later = torch.cat([keep[:, 1:], torch.ones_like(keep[:, :1])], 1)
    g = _running(later.flip(1), g.flip(1)).flip(1)
    got["db"] = (g * split(step * u)[..., None]).sum(3).to(y.dtype)
    into = (g * b).sum(4).flatten(2)  # the gradient of step * u
    got["du"] = (into * step + dy * s["skip"]).to(y.dtype)
    got["dskip"] = (dy * u).sum((0, 1), dtype=torch.float64).float()
    # through the decay: h[t - 1] decay[t] g[t] is the gradient of step * a
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    through = (g * before * keep).flatten(2, 3)
    got["da_log"] = (through * step[..., None]).sum((0, 1), dtype=torch.float64).mul(a).float()
    dstep = (through * a).sum(3) + into * u
    draw_ = dstep * torch.sigmoid(raw)
    if s["lengths"] is not None:
        draw_ = draw_ * _counts(s, draw_.shape[1])
    got["ddt"] = draw_.to(y.dtype)
    got["ddt_bias"] = draw_.sum((0, 1), dtype=torch.float64).float()
    return got


def _plain_sample(s):
    """Words in descending order, equal ones in that of their numbers: the first top_k, of these the fewest whose
    share reaches top_p, of these the ones at least min_p times as likely as the first; then, in the order of their
    numbers, the first whose running sum passes uniform times their total."""
    rows, words = s["logits"].shape
    col = lambda v, kind: (v if torch.is_tensor(v) else torch.full((rows,), v, device="cuda", dtype=kind))[:, None]  # noqa: E731
    temperature = col(s["set"]["temperature"], torch.float64).double()
    top_k = col(s["set"]["top_k"], torch.int64).long()
    top_p, min_p = (col(s["set"][k], torch.float64).double() for k in ("top_p", "min_p"))
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    greedy = temperature <= 0
    weight = torch.exp((x - top) / torch.where(greedy, 1.0, temperature))
    falling, order = torch.sort(x, dim=1, descending=True, stable=True)
    sorted_weight = torch.gather(weight, 1, order)
    place = torch.arange(words, device="cuda")[None]
    sorted_weight = sorted_weight * ((top_k <= 0) | (place < top_k))
    upto = torch.cumsum(sorted_weight, 1)
    kept = (top_p >= 1) | (place == 0) | (upto - sorted_weight < top_p * upto[:, -1:])
    kept &= (sorted_weight >= min_p) & (place < torch.where(greedy, 1, words))
    weight = torch.zeros_like(weight).scatter_(1, order, sorted_weight * kept)
    upto = torch.cumsum(weight, 1)
    passed = (upto > s["uniform"].double()[:, None] * upto[:, -1:]) & (weight > 0)
    token = passed.to(torch.uint8).argmax(1)
    return torch.where(falling[:, 0] > -math.inf, token, -1).to(torch.int32)


# ----------------------------------------------------------------- the operators
def _own_conv(s):
    from dlvk_b200.ops import ssm

    op, silu = s["case"]["op"], s["case"]["silu"]
    if op == "conv_step":
        y = ssm.short_conv_step(s["x"], s["weight"], s["bias"], s["state"], silu=silu, out_state=s["next"])
        return {"y": y, "state": s["next"]}
    if op == "conv_prompt":
        y, state = ssm.short_conv_fwd(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"],
                                      silu=silu, want_state=True)
        return {"y": y, "state": state}
    y, _ = ssm.short_conv_fwd(s["x"], s["weight"], s["bias"], lengths=s["lengths"], silu=silu)
    dx, dweight, dbias = ssm.short_conv_bwd(s["x"], s["weight"], s["bias"], s["dy"], lengths=s["lengths"], silu=silu)
    got = {"y": y, "dx": dx, "dweight": dweight}
    if dbias is not None:
        got["dbias"] = dbias
    return got


def _own_scan(s):
    from dlvk_b200.ops import ssm

    op = s["case"]["op"]
    args = (s["u"], s["dt"], s["a_log"], s["b"], s["c"])
    more = {"skip": s["skip"], "z": s["z"], "dt_bias": s["dt_bias"]}
    if op == "scan_step":
        y = ssm.state_scan_step(*args, s["state"], out_state=s["next"], **more)
        return {"y": y, "state": s["next"]}
    if op == "scan_prompt":
        y, state, _ = ssm.state_scan_fwd(*args, state=s["state"], lengths=s["lengths"], want_state=True, **more)
        return {"y": y, "state": state}
    y, _, saved = ssm.state_scan_fwd(*args, lengths=s["lengths"], save=True, **more)
    grads = ssm.state_scan_bwd(*args, dy=s["dy"], saved=saved, lengths=s["lengths"], **more)
    got = {"y": y}
    got.update((k, v) for k, v in grads._asdict().items() if v is not None)
    return got


def _own_sample(s):
    from dlvk_b200.ops import sampling

    return sampling.sample_tokens(s["logits"], s["uniform"], **s["set"])


def run(s):
    kind = s["case"]["op"].split("_")[0]
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "sample": _own_sample}[kind](s)
    return {"conv": _plain_conv, "scan": _plain_scan, "sample": _plain_sample}[kind](s)


# ------------------------------------------------------------------------ the work
def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["words"]
        return {"bytes": n * _TYPES[case["dtype"]].itemsize + 8 * case["rows"], "flops": 4 * n}
    size = _TYPES[case["dtype"]].itemsize
    b, t, d = case["batch"], case["tokens"], case["channels"]
    n = b * t * d
    if case["op"].startswith("conv"):
        k = case["taps"]
        params = 4 * d * (k + 1)
        if case["op"] == "conv_train":  # x and dy in, y and dx out
            return {"bytes": 4 * size * n + 2 * params, "flops": 6 * k * n}
        state = size * b * (k - 1) * d
        return {"bytes": 2 * size * n + params + state * (2 if case["state"] else 1), "flops": 2 * k * n}
    st, gates = case["states"], 1 if case["gate"] else 0
    params = 4 * d * (st + 2)
    rows = 2 * size * b * t * case["groups"] * st
    if case["op"] == "scan_train":  # u, dt, z, dy, b, c in; y and all their gradients out
        return {"bytes": size * n * (6 + 2 * gates) + 2 * rows + 2 * params, "flops": 24 * n * st}
    state = 4 * b * d * st
    return {"bytes": size * n * (3 + gates) + rows + params + state * (2 if case["state"] else 1),
            "flops": 7 * n * st}


# --------------------------------------------------------------- values in 64 bits
def _exact_conv(s):
    case = s["case"]
    x = (s["x"] if s["x"].dim() == 3 else s["x"][:, None]).double()
    k, tokens = s["weight"].shape[1], x.shape[1]
    w = s["weight"].double()
    bias = s["bias"].double() if s["bias"] is not None else None
    train = case["op"] == "conv_train"
    leaves = [v.requires_grad_(train) for v in (x, w, bias) if v is not None]
    counted = None
    y = 0.0
    if s["lengths"] is not None:
        counted = torch.arange(tokens, device="cuda")[None, :, None] < s["lengths"][:, None, None]
    state = s["state"].double() if s["state"] is not None else x.new_zeros(x.shape[0], k - 1, x.shape[2])
    whole = torch.cat([state, x], 1)
    for j in range(k):
        y = y + w[:, j] * whole[:, j:j + tokens]
    y = y + bias if bias is not None else y
    y = y / (1 + torch.exp(-y)) if case["silu"] else y
    y = y * counted if counted is not None else y
    if train:
        grads = torch.autograd.grad(y, leaves, s["dy"].double())
        return dict(zip(["y", "dx", "dweight", "dbias"], [y.detach(), *grads]))
    if case["op"] == "conv_step":
        return {"y": y[:, 0], "state": whole[:, 1:]}
    ends = s["lengths"].tolist() if s["lengths"] is not None else [tokens] * x.shape[0]
    return {"y": y, "state": torch.stack([whole[i, e:e + k - 1] for i, e in enumerate(ends)])}


def _exact_scan(s):
    case = s["case"]
    train = case["op"] == "scan_train"
    one = s["u"].dim() == 2
    wide = lambda v: None if v is None else (v[:, None] if one else v).double().requires_grad_(train)  # noqa: E731
    named = {"u": wide(s["u"]), "dt": wide(s["dt"]), "b": wide(s["b"]), "c": wide(s["c"]), "z": wide(s["z"])}
    for k in ("a_log", "skip", "dt_bias"):
        named[k] = s[k].double().requires_grad_(train)
    batch, tokens, channels = named["u"].shape
    per = channels // case["groups"]
    rate = torch.exp(named["a_log"])
    h = s["state"].double() if s["state"] is not None else rate.new_zeros(batch, channels, case["states"])
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((batch,), tokens, device="cuda")
    out = []
    with torch.set_grad_enabled(train):
        step = torch.logaddexp(named["dt"] + named["dt_bias"], torch.zeros((), device="cuda", dtype=torch.float64))
        for t in range(tokens):
            here = (lengths > t)[:, None, None]
            bt = named["b"][:, t].repeat_interleave(per, 1)
            new = h * torch.exp(-step[:, t, :, None] * rate) + (step[:, t] * named["u"][:, t])[..., None] * bt
            h = torch.where(here, new, h)
            yt = torch.matmul(h.unflatten(1, (case["groups"], per)), named["c"][:, t][..., None])[..., 0].flatten(1)
            out.append((yt + named["skip"] * named["u"][:, t]) * here[..., 0])
        y = torch.stack(out, 1)
        if named["z"] is not None:
            y = y * named["z"] / (1 + torch.exp(-named["z"]))
    if case["op"] == "scan_prompt":
        return {"y": y, "state": h}
    if case["op"] == "scan_step":
        return {"y": y[:, 0], "state": h}
    names = [k for k, v in named.items() if v is not None]
    grads = torch.autograd.grad(y, [named[k] for k in names], s["dy"].double())
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def exact(case, seed):
    if case["op"] == "sample":
        return None  # numbers of words
    s = prepare(case, seed)
    return _exact_conv(s) if case["op"].startswith("conv") else _exact_scan(s)
