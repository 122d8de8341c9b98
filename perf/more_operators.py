"""The operators that answer with the text model in 8-bit integers, as cases to measure: rows normalised and quantised with a
scale each, matrix products of such rows with int8 weights, and the choice of a token from the logits.

``run`` computes a case in plain torch operations or, with ``own`` set, through the package's operators.

Rows.  ``h = x + residual``; ``y`` is h, its RMSNorm (``weight``) or its LayerNorm (``weight`` and ``bias``), divided by
``smooth`` where there is one; ``scale = max |y| / 127``, ``code = round(y / scale)``.  The values that codes stand for come back
in x's type, beside the scales and h in x's type.

Products.  ``y[m, n] = scale[m] wscale[n] sum_k code[m, k] weight[n, k] + bias[n] + residual[m, n]``; a gated one has 2 N weight
rows, the gate's first, and gives ``silu(gate) * up``.

Tokens.  Of the logits l of a row, ``w_i = round(2^44 exp((l_i - max l) / temperature))``, whole numbers.  Kept are the
``top_k`` largest logits (0: all) with ``w_i >= min_p 2^44``, of these the most likely ones up to the one with which their sum
reaches ``top_p`` of it; equal logits go by index.  The token is the first, by index, up to which the kept w add up to more than
``floor(u sum w)``; its log-probability among the kept comes with it.  Temperature 0 takes the largest logit.
"""

import math
import random

import torch

own = False

UNIT = 2.0 ** 44  # the weight of the most likely token
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- cases

def _rows(name=None, *, dtype="bf16", m=1, k=960, norm="rms", residual=True, smooth=False):
    c = {"op": "rows", "dtype": dtype, "m": m, "k": k, "norm": norm, "residual": residual, "smooth": smooth}
    return c | ({"name": name} if name else {})


def _product(name=None, *, dtype="bf16", m=1, n=960, k=960, gated=False, bias=False, residual=False):
    c = {"op": "product", "dtype": dtype, "m": m, "n": n, "k": k, "gated": gated, "bias": bias, "residual": residual}
    return c | ({"name": name} if name else {})


def _tokens(name=None, *, dtype="fp32", batch=1, vocab=49280, temperature=(0.7, 0.7), top_k=(0, 0), top_p=(1.0, 1.0),
            min_p=(0.0, 0.0), masked=0.0, spread=2.5):
    """Every row has its own settings, spread between the two of each pair; ``masked``: the share of logits at -infinity;
    ``spread``: the logits' standard deviation."""
    c = {"op": "tokens", "dtype": dtype, "batch": batch, "vocab": vocab, "masked": masked, "spread": spread}
    for key, (low, high) in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        c |= {key + "_min": low, key + "_max": high}
    return c | ({"name": name} if name else {})


def listed():
    return [
        # one robot's next token on its way into a layer: the smallest call
        _rows("rows one", m=1, k=960),
        # the prompts of 64 robots (two images, language, state) on their way into a layer
        _rows("rows prompts", m=64 * 177, k=960),
        # the same prompts between the two products of the feed-forward block: no norm, smoothed channels
        _rows("rows smoothed", m=64 * 177, k=2560, norm="none", residual=False, smooth=True),
        # a wider model with LayerNorm
        _rows("rows wide", dtype="fp16", m=8192, k=4096, norm="layer"),
        # one robot's next token: queries, keys and values in one product
        _product("product one", m=1, n=1600, k=960),
        # the logits of 64 sequences' next tokens, over the whole vocabulary
        _product("product logits", dtype="fp32", m=64, n=49280, k=960),
        # gate and up projections of the prompts of 64 robots
        _product("product gated", m=64 * 177, n=2560, k=960, gated=True),
        # the second product of a wider model's feed-forward block, added to the hidden states
        _product("product wide", dtype="fp16", m=8192, n=4096, k=11008, residual=True),
        # one sequence's next token
        _tokens("tokens one", batch=1, temperature=(0.7, 0.7), top_k=(50, 50), top_p=(0.95, 0.95)),
        # a server's batch, every request with settings of its own, some of them greedy
        _tokens("tokens mixed", batch=256, temperature=(0.0, 1.3), top_k=(0, 200), top_p=(0.5, 1.0), min_p=(0.0, 0.1)),
        # many sequences drawn from the whole distribution, as rollouts for training are
        _tokens("tokens all", dtype="bf16", batch=512, temperature=(1.0, 1.0)),
        # a large vocabulary of which a grammar forbids a half, with a high temperature: top_p keeps thousands
        _tokens("tokens large", dtype="bf16", batch=64, vocab=131072, temperature=(1.0, 1.5), top_p=(0.9, 0.99), masked=0.5,
                spread=1.5),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _range(rng, low, high):
    a, b = rng.uniform(low, high), rng.uniform(low, high)
    return rng.choice([(a, a), (min(a, b), max(a, b))])


def draw(rng):
    op = rng.choice(["rows", "product", "tokens"])
    if op == "rows":
        k = rng.choice([720, 768, 960, 2048, 2560, 4096, _spread(rng, 16, 16384)])
        return _rows(dtype=rng.choice(["bf16", "bf16", "fp16"]), m=_spread(rng, 1, min(32768, 33500000 // k)), k=k,
                     norm=rng.choice(["rms", "rms", "layer", "none"]), residual=rng.random() < 0.6, smooth=rng.random() < 0.4)
    if op == "product":
        k = rng.choice([720, 768, 960, 2048, 2560, 4096, _spread(rng, 16, 11008)])
        n = rng.choice([960, 1600, 720, 2560, 4096, _spread(rng, 16, 16384)])
        gated = rng.random() < 0.3
        m = _spread(rng, 1, max(1, min(16384, int(1.5e11 / (k * n)))))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return _product(dtype=dtype, m=m, n=n, k=k, gated=gated, bias=not gated and rng.random() < 0.4,
                        residual=not gated and rng.random() < 0.4)
    vocab = rng.choice([256, 32000, 49280, 49280, 131072, _spread(rng, 2, 200000)])
    batch = _spread(rng, 1, max(1, min(512, 12000000 // vocab)))
    top_k = rng.choice([(0, 0), (0, 0), (1, 100), (_spread(rng, 1, vocab),) * 2])
    return _tokens(dtype=rng.choice(["fp32", "bf16", "fp16"]), batch=batch, vocab=vocab, temperature=_range(rng, 0.2, 2.0),
                   top_k=top_k, top_p=rng.choice([(1.0, 1.0), _range(rng, 0.3, 1.0)]),
                   min_p=rng.choice([(0.0, 0.0), _range(rng, 0.0, 0.2)]), masked=rng.choice([0.0, 0.0, 0.3, 0.9]),
                   spread=rng.choice([1.0, 2.5, 4.0]))


# ----------------------------------------------------------------------------- inputs

def _codes(gen, rows, k):
    """int8 rows as quantising leaves them: normal values of which the largest is near 127, rows 16 bytes apart."""
    x = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
    x[:, :k] = torch.randn(rows, k, generator=gen, device="cuda").mul_(36).round_().clamp_(-127, 127)
    return x[:, :k]


def _uniform(gen, n, low, high):
    return torch.rand(n, generator=gen, device="cuda") * (high - low) + low


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, state = TYPES[case["dtype"]], {"case": dict(case)}

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "rows":
        m, k = case["m"], case["k"]
        x = normal(m, k)
        x[:, k // 5 :: k // 4 + 1] *= 6.0  # a few channels of larger size, as a model's hidden states have them
        state |= {"x": x.to(dtype), "residual": None, "weight": None, "bias": None, "smooth": None, "eps": 1e-5}
        if case["residual"]:
            state["residual"] = (2.0 * normal(m, k)).to(dtype)
        if case["norm"] != "none":
            state["weight"] = (1.0 + 0.2 * normal(k)).to(dtype)
        if case["norm"] == "layer":
            state["bias"] = (0.1 * normal(k)).to(dtype)
        if case["smooth"]:
            state["smooth"] = torch.exp(0.5 * normal(k))
        return state
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        rows = 2 * n if case["gated"] else n
        state |= {"codes": _codes(gen, m, k), "scale": _uniform(gen, m, 0.01, 0.05), "weight": _codes(gen, rows, k),
                  "wscale": _uniform(gen, rows, 0.5, 1.5) * (0.02 / math.sqrt(k)), "bias": None, "residual": None}
        if case["bias"]:
            state["bias"] = 0.1 * normal(n)
        if case["residual"]:
            state["residual"] = normal(m, n).to(dtype)
        return state
    batch, vocab = case["batch"], case["vocab"]
    x = normal(batch, vocab) * case["spread"]
    likely = torch.randint(vocab, (batch, 8), generator=gen, device="cuda")
    x.scatter_add_(1, likely, normal(batch, 8).abs() * 3.0 + 6.0)
    if case["masked"]:
        hidden = torch.rand(batch, vocab, generator=gen, device="cuda") < case["masked"]
        hidden.scatter_(1, likely, False)
        x.masked_fill_(hidden, -math.inf)
    state["logits"] = x.to(dtype)
    state["u"] = torch.rand(batch, generator=gen, device="cuda")
    for key in ("temperature", "top_k", "top_p", "min_p"):
        value = _uniform(gen, batch, case[key + "_min"], case[key + "_max"])
        state[key] = value.to(torch.int32) if key == "top_k" else value
    # where settings begin at 0, a quarter of the rows has exactly that
    if case["temperature_min"] == 0:
        state["temperature"][::4] = 0
    if case["top_k_min"] == 0:
        state["top_k"][1::4] = 0
    return state


# ----------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"rows": _own_rows, "product": _own_product, "tokens": _own_tokens}[op](state)
    return {"rows": _plain_rows, "product": _plain_product, "tokens": _plain_tokens}[op](state)


def _own_rows(s):
    from smolvla_mujoco_libero_b200 import ops
    r = ops.quantize_rows(s["x"], weight=s["weight"], bias=s["bias"], eps=s["eps"], residual=s["residual"], smooth=s["smooth"],
                          want_values=True)
    return {"values": r.values, "scale": r.scale, "sum": r.sum if s["residual"] is not None else None}


def _own_product(s):
    from smolvla_mujoco_libero_b200 import ops
    return ops.linear_i8_rows(s["codes"], s["scale"], s["weight"], s["wscale"], bias=s["bias"], residual=s["residual"],
                              gated=s["case"]["gated"], dtype=TYPES[s["case"]["dtype"]])


def _own_tokens(s):
    from smolvla_mujoco_libero_b200 import ops
    tokens, logprob = ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                        min_p=s["min_p"])
    return {"tokens": tokens, "logprob": logprob}


def _plain_rows(s):
    x, residual = s["x"], s["residual"]
    y = x.float()
    if residual is not None:
        y = y + residual.float()
    total = y.to(x.dtype) if residual is not None else None
    if s["bias"] is not None:
        y = y - y.mean(-1, keepdim=True)
    if s["weight"] is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["smooth"] is not None:
        y = y / s["smooth"]
    scale = y.abs().amax(-1) / torch.full((), 127.0, device=x.device)  # a tensor: a number would be multiplied by its reciprocal
    codes = torch.where(scale[:, None] > 0, torch.round(y / scale[:, None]), 0.0).clamp(-127, 127)
    return {"values": (codes * scale[:, None]).to(x.dtype), "scale": scale, "sum": total}


def _plain_product(s):
    case = s["case"]
    y = torch.matmul(s["codes"].float(), s["weight"].float().T).mul_(s["scale"][:, None]).mul_(s["wscale"])
    if case["gated"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    if s["bias"] is not None:
        y += s["bias"]
    if s["residual"] is not None:
        y += s["residual"].float()
    return y.to(TYPES[case["dtype"]])


def _plain_tokens(s):
    x = s["logits"].double()
    greedy = s["temperature"] == 0
    temperature = torch.where(greedy, 1.0, s["temperature"]).double()
    top_k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], x.shape[1]))
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    value, index = order.values, order.indices
    w = torch.round(torch.exp((value - value[:, :1]) / temperature[:, None]) * UNIT).long()
    rank = torch.arange(x.shape[1], device=x.device)
    first = rank == 0
    kept = (rank < top_k[:, None]) & ((w.double() >= (s["min_p"].double() * UNIT)[:, None]) | first)
    w = torch.where(kept, w, 0)
    before = w.cumsum(-1) - w
    limit = torch.ceil(s["top_p"].double() * w.sum(-1).double()).long()
    kept = kept & ((before < limit[:, None]) | first | (s["top_p"] >= 1)[:, None])
    by_index = torch.zeros_like(w).scatter_(1, index, torch.where(kept, w, 0))
    upto = by_index.cumsum(-1)
    total = upto[:, -1]
    target = torch.minimum((s["u"].double() * total.double()).long(), total - 1)
    token = torch.searchsorted(upto, target[:, None], right=True)
    logprob = torch.log(by_index.gather(1, token).squeeze(1).double() / total.double())
    return {"tokens": token.squeeze(1).int(), "logprob": logprob.float()}


# ----------------------------------------------------------------------------- work and the exact answer

def work(case):
    if case["op"] == "rows":
        # x in, codes and values out; with a residual also that in and the sum out
        size = case["m"] * case["k"]
        per = 2 + 1 + 2 + (4 if case["residual"] else 0)
        return {"bytes": size * per + 4 * case["m"], "flops": 8 * size}
    if case["op"] == "product":
        m, n, k, rows = case["m"], case["n"], case["k"], case["n"] * (2 if case["gated"] else 1)
        out = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": m * k + rows * (k + 4) + 4 * m + m * n * out * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * rows * k}
    size = case["batch"] * case["vocab"]
    return {"bytes": size * (4 if case["dtype"] == "fp32" else 2) + 28 * case["batch"], "flops": size}


def _exact_rows(case, s):
    h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    y = h
    if case["norm"] == "rms":
        y = h / (h.pow(2).sum(-1, keepdim=True) / case["k"] + s["eps"]).sqrt() * s["weight"].double()
    elif case["norm"] == "layer":
        var, mean = torch.var_mean(h, -1, correction=0, keepdim=True)
        y = (h - mean) / (var + s["eps"]).sqrt() * s["weight"].double() + s["bias"].double()
    if case["smooth"]:
        y = y / s["smooth"].double()
    largest = torch.maximum(y.max(-1, keepdim=True).values, -y.min(-1, keepdim=True).values)
    steps = torch.where(largest > 0, y * 127 / largest, 0.0)
    return {"values": steps.round() * largest / 127, "scale": largest.squeeze(1) / 127, "sum": h if case["residual"] else None}


def _exact_product(case, s):
    parts, n = [], case["n"]
    weight = s["weight"].double().T
    for a in range(0, case["m"], 2048):
        y = s["codes"][a:a + 2048].double() @ weight
        y = torch.einsum("mn,m,n->mn", y, s["scale"][a:a + 2048].double(), s["wscale"].double())
        if case["gated"]:
            y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
        parts.append(y)
    y = torch.cat(parts)
    if case["bias"]:
        y = y + s["bias"].double()
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_logprob(case, s):
    """Row by row from the definition, the most likely tokens first; None where that would take long."""
    if case["batch"] > 1024:
        return None
    found = []
    for b in range(case["batch"]):
        x = s["logits"][b].double()
        if s["temperature"][b] == 0:
            found.append(0.0)
            continue
        p = torch.exp((x - x.max()) / s["temperature"][b].double())
        p = torch.floor(p * 2 ** 44 + 0.5) / 2 ** 44
        # lexicographic: by falling logit, then by rising index
        order = torch.argsort(-x, stable=True)
        k = int(s["top_k"][b])
        order = order[:k] if k > 0 else order
        alive = int((p[order] >= float(s["min_p"][b])).sum())
        order = order[:max(1, alive)]
        mass = p[order]
        if s["top_p"][b] < 1:
            share = (torch.cumsum(mass, 0) - mass) / mass.sum()
            order = order[:max(1, int((share < float(s["top_p"][b])).sum()))]
        order = order.sort().values
        mass = p[order]
        place = torch.searchsorted(torch.cumsum(mass, 0), (s["u"][b].double() * mass.sum()).reshape(1), right=True)
        found.append(float(torch.log(mass[min(int(place), len(mass) - 1)] / mass.sum())))
    return torch.tensor(found, dtype=torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        return _exact_rows(case, s)
    if case["op"] == "product":
        return _exact_product(case, s)
    return {"tokens": None, "logprob": _exact_logprob(case, s)}
