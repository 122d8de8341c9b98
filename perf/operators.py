"""The serving operators of the text model as cases to measure: attention over packed prompts, appending to a paged
key/value cache with the position rotation, and attention over such a cache.

``run`` computes a case in plain torch operations (fp32) or, with ``own`` set, through the package's operators.

Cache pages.  A cache is one tensor of pages; sequence b keeps its entry n in page ``page_table[b, n // page]``, slot
``n % page``.  16 bits: ``[pages, kv_heads, 2, page, dim]`` (keys, then values).  4 bits: uint8 ``[pages, kv_heads,
page, dim + dim / 4]``, of which each kv head's bytes are key codes ``[page, dim / 2]``, value codes, then for keys and
for values bf16 (step, low) ``[page, dim / 32, 2]``; a value is ``low + step * code``, dimension 2 j in the low half of byte j.
"""

import math
import random

import torch

own = False

GROUP = 32            # dimensions that share a (step, low) pair in a 4-bit cache
WAVELENGTH = 10000.0  # of the position rotation
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ----------------------------------------------------------------------------- cases

def _case(op, name=None, *, dtype="bf16", batch=1, new=(1, 1), past=(0, 0), heads=(15, 5, 64), causal=True, bits=16,
          page=16, pattern=1):
    """``new`` tokens per sequence after ``past`` ones, both ranges of lengths; ``pattern`` seeds the lengths."""
    c = {"op": op, "dtype": dtype, "batch": batch, "new_min": new[0], "new_max": new[1], "past_min": past[0],
         "past_max": past[1], "hq": heads[0], "hkv": heads[1], "dim": heads[2], "pattern": pattern}
    c |= {"causal": causal} if op == "packed" else {"bits": bits, "page": page}
    return c | ({"name": name} if name else {})


TEXT = (15, 5, 64)    # the text model's heads
WIDE = (32, 8, 128)   # a wider text model


def listed():
    return [
        # one robot's prefix (two images, language, state) prefilled alone: latency counts
        _case("packed", "prompt one", new=(177, 177), heads=TEXT),
        # a server's batch: prompts of 1 to 1024 tokens, some after a prefix that is already there
        _case("packed", "prompts ragged", dtype="fp16", batch=64, new=(1, 1024), past=(0, 300), heads=TEXT),
        # one long history
        _case("packed", "prompt long", new=(16384, 16384), heads=TEXT),
        # several long prompts of a wider model
        _case("packed", "prompts wide", batch=4, new=(1024, 4096), heads=WIDE),
        # one robot's next token: the smallest call
        _case("append", "append one", past=(177, 177), heads=TEXT),
        # one token of each of 256 sequences into a 4-bit cache
        _case("append", "append step 4 bits", batch=256, past=(177, 4096), heads=TEXT, bits=4),
        # whole prompts into a 16-bit cache
        _case("append", "append prompts", dtype="fp16", batch=32, new=(64, 2048), past=(0, 100), heads=TEXT, page=64),
        # whole prompts of a wider model into a 4-bit cache
        _case("append", "append prompts 4 bits", batch=16, new=(512, 4096), heads=WIDE, bits=4, page=32),
        # one robot's next token over its prefix
        _case("paged", "decode one", past=(177, 177), heads=TEXT, bits=4),
        # the next token of 64 sequences of different ages
        _case("paged", "decode many", batch=64, past=(255, 8191), heads=TEXT, bits=4),
        # five drafted tokens of each of 24 sequences over a 16-bit cache
        _case("paged", "drafts 16 bits", dtype="fp16", batch=24, new=(5, 5), past=(100, 4000), heads=TEXT, page=32),
        # two very long histories of a wider model
        _case("paged", "decode long", batch=2, past=(100000, 131071), heads=WIDE, bits=4, page=64),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["packed", "append", "paged"])
    heads = rng.choice([TEXT, WIDE, (12, 12, 64), (16, 2, 64), (8, 1, 128), (6, 3, 128), (14, 2, 64), (24, 8, 128)])
    pattern, dtype = rng.randrange(1 << 20), rng.choice(["bf16", "bf16", "fp16"])
    if op == "packed":
        batch = _spread(rng, 1, 128)
        # batch * heads * longest^2 stays below a quarter of the long prompt's
        top = max(1, min(8192, int(math.sqrt(1.0e9 / (batch * heads[0])))))
        new = _spread(rng, 1, top)
        past = rng.choice([0, 0, _spread(rng, 1, max(1, min(top, 2000)))])
        return _case("packed", dtype=dtype, batch=batch, new=(_spread(rng, 1, new), new), past=(0, past), heads=heads,
                     causal=rng.random() < 0.8, pattern=pattern)
    bits, page = rng.choice([4, 4, 16]), rng.choice([16, 16, 32, 48, 64, 128])
    if op == "append":
        batch = _spread(rng, 1, 512)
        new = rng.choice([1, _spread(rng, 1, max(1, min(4096, 24000 // batch)))])
        past = _spread(rng, 1, max(1, min(4096, 200000 // batch)))
        return _case("append", dtype=dtype, batch=batch, new=(rng.choice([1, new]), new), past=(0, past), heads=heads,
                     bits=bits, page=page, pattern=pattern)
    batch = _spread(rng, 1, 256)
    new = rng.choice([1, 1, 1, rng.randrange(2, 9)])
    past = _spread(rng, 1, max(1, min(100000, 2500000 // (batch * heads[1] * heads[2] // 64) // new)))
    return _case("paged", dtype=dtype, batch=batch, new=(rng.choice([1, new]), new), past=(rng.randrange(0, past + 1), past),
                 heads=heads, bits=bits, page=page, pattern=pattern)


def _lengths(case):
    """New tokens and earlier tokens of each sequence, from the case alone."""
    rng = random.Random(case["pattern"])
    new = [_spread(rng, case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    past = [rng.randrange(case["past_min"], case["past_max"] + 1) for _ in range(case["batch"])]
    return new, past


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


# ----------------------------------------------------------------------------- inputs

def _rows(gen, rows, heads, dim, outliers=False):
    """Activations: normal, and for keys a few channels of larger size, as projections without a norm give them."""
    x = torch.randn(rows, heads, dim, generator=gen, device="cuda")
    if outliers:
        x[..., dim // 5 :: dim // 4] *= 3.0
    return x


def _quantise(x):
    """(codes, step, low) of groups of 32 of the last dimension.  The quotients are true divisions: a value that lies
    halfway between two codes (16-bit values often do) is then halfway in any precision."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    fifteen = torch.full((), 15.0, device=x.device)  # a tensor: division by a number multiplies by its reciprocal
    step = ((high - low) / fifteen).to(torch.bfloat16)
    low = low.to(torch.bfloat16)
    s, m = step.float(), low.float()
    codes = torch.where(s > 0, torch.round((g - m) / s), 0.0).clamp(0, 15)
    return codes.flatten(-2), step.squeeze(-1), low.squeeze(-1)


def _values(codes, step, low):
    """What codes stand for, in the codes' type."""
    g = codes.unflatten(-1, (-1, GROUP))
    return (g * step.unsqueeze(-1).to(g.dtype) + low.unsqueeze(-1).to(g.dtype)).flatten(-2)


def _packed_bytes(codes):
    c = codes.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _parts(data, page, dim):
    """Views of a 4-bit cache: key codes, value codes, key (step, low), value (step, low)."""
    n, g = page * dim // 2, page * dim // GROUP * 4
    data = data.flatten(-2)
    codes = [data[..., i * n : (i + 1) * n].unflatten(-1, (page, dim // 2)) for i in (0, 1)]
    pairs = [data[..., 2 * n + i * g : 2 * n + (i + 1) * g].view(torch.bfloat16).unflatten(-1, (page, dim // GROUP, 2))
             for i in (0, 1)]
    return codes + pairs


def _cache(case, gen, pages):
    dtype, page, dim, hkv = TYPES[case["dtype"]], case["page"], case["dim"], case["hkv"]
    if case["bits"] == 16:
        data = torch.empty(pages, hkv, 2, page, dim, dtype=dtype, device="cuda")
        data[:, :, 0] = _rows(gen, pages * hkv, page, dim, outliers=True).view(pages, hkv, page, dim).to(dtype)
        data[:, :, 1] = _rows(gen, pages * hkv, page, dim).view(pages, hkv, page, dim).to(dtype)
        return data
    data = torch.empty(pages, hkv, page, dim + dim // 4, dtype=torch.uint8, device="cuda")
    parts = _parts(data, page, dim)
    for i in (0, 1):
        x = _rows(gen, pages * hkv, page, dim, outliers=i == 0).view(pages, hkv, page, dim)
        codes, step, low = _quantise(x)
        parts[i].copy_(_packed_bytes(codes))
        parts[2 + i].copy_(torch.stack([step, low], -1))
    return data


def _rotation(positions, dim):
    """(cos, sin) of every position and pair of dimensions, from angles in 64 bits."""
    inv = WAVELENGTH ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, past = _lengths(case)
    total = [n + p for n, p in zip(new, past)]
    dtype, hq, hkv, dim = TYPES[case["dtype"]], case["hq"], case["hkv"], case["dim"]
    state = {"case": dict(case), "cu_q": _ints(_starts(new)), "new_longest": max(new), "longest": max(total),
             "scale": dim ** -0.5}
    if case["op"] == "packed":
        state["cu_k"] = _ints(_starts(total))
        kv = torch.cat([_rows(gen, sum(total), hkv, dim, outliers=True), _rows(gen, sum(total), hkv, dim)], 1).to(dtype)
        q = _rows(gen, sum(new), hq, dim).to(dtype)
        if not any(past):  # all three are parts of one projection's output, as a layer has them
            q, kv = torch.cat([q, kv], 1).split([hq, 2 * hkv], 1)
        state |= {"q": q, "k": kv[:, :hkv], "v": kv[:, hkv:]}
        return state
    per = [-(-n // case["page"]) for n in total]
    pages = sum(per) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in per:
        table.append(order[at : at + n] + [0] * (max(per) - n))
        at += n
    state |= {"kv_len": _ints(total), "page_table": _ints(table), "cache": _cache(case, gen, pages)}
    if case["op"] == "append":
        qkv = torch.cat([_rows(gen, sum(new), hq, dim), _rows(gen, sum(new), hkv, dim, outliers=True),
                         _rows(gen, sum(new), hkv, dim)], 1).to(dtype)
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        state |= {"q": q, "k": k, "v": v, "rope": _rotation(max(total), dim)}
    else:
        state["q"] = _rows(gen, sum(new), hq, dim).to(dtype)
    return state


# ----------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"packed": _own_packed, "append": _own_append, "paged": _own_paged}[op](state)
    return {"packed": _plain_packed, "append": _plain_append, "paged": _plain_paged}[op](state)


def _own_packed(s):
    from smolvla_mujoco_libero_b200 import ops
    return ops.packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"])


def _own_append(s):
    from smolvla_mujoco_libero_b200 import ops
    if s["case"]["bits"] == 16:
        q = ops.kv_append(s["cache"], s["k"], s["v"], s["cu_q"], s["kv_len"], s["page_table"], q=s["q"], rope_cs=s["rope"])
        return {"q": q, "cache": s["cache"]}
    # the rows as the cache holds them come back too: prompt attention reads them
    q, k, v = ops.kv_append(s["cache"], s["k"], s["v"], s["cu_q"], s["kv_len"], s["page_table"], q=s["q"],
                            rope_cs=s["rope"], want_rows=True)
    return {"q": q, "k": k, "v": v}


def _own_paged(s):
    from smolvla_mujoco_libero_b200 import ops
    return ops.paged_attention(s["q"], s["cache"], s["cu_q"], s["kv_len"], s["page_table"])


def _tokens(s, rows):
    """Sequence of every token, and its place there."""
    t = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu_q"], t, right=True) - 1
    return seq, t - s["cu_q"][seq]


def _attend(s, q, k, v, lq, lk, causal):
    """Attention of q [B, Lq, hq, D] over k, v [B, Lk, hkv, D], all fp32 and padded; lq, lk: the lengths."""
    batch, longest, hq, dim = q.shape
    keys, hkv = k.shape[1], k.shape[2]
    g = hq // hkv
    q = q.view(batch, longest, hkv, g, dim).permute(0, 2, 3, 1, 4).reshape(batch, hkv, g * longest, dim)
    p = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(s["scale"]).view(batch, hkv, g, longest, keys)
    j = torch.arange(keys, device="cuda")
    if causal:
        end = (lk - lq)[:, None] + torch.arange(longest, device="cuda") + 1
        hidden = j >= torch.minimum(end, lk[:, None])[:, :, None]
    else:
        hidden = (j >= lk[:, None])[:, None, :].expand(batch, longest, keys)
    p.masked_fill_(hidden[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch, hkv, g * longest, keys), v.permute(0, 2, 1, 3)).view(batch, hkv, g, longest, dim)
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, longest, hq, dim)


def _padded(x, starts, longest):
    at = (starts[:-1, None] + torch.arange(longest, device="cuda")).clamp_(max=x.shape[0] - 1)
    return x[at].float()


def _plain_packed(s):
    q, cu_q, cu_k = s["q"], s["cu_q"], s["cu_k"]
    o = _attend(s, _padded(q, cu_q, s["new_longest"]), _padded(s["k"], cu_k, s["longest"]),
                _padded(s["v"], cu_k, s["longest"]), cu_q.diff(), cu_k.diff(), s["case"]["causal"])
    return o[_tokens(s, q.shape[0])].to(q.dtype)


def _rotate(x, cs):
    """x [T, heads, D] fp32; cs [T, D / 2, 2]."""
    x1, x2 = x.chunk(2, -1)
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([x1 * c - x2 * n, x2 * c + x1 * n], -1)


def _plain_append(s):
    case, page, dim = s["case"], s["case"]["page"], s["case"]["dim"]
    dtype = s["q"].dtype
    seq, i = _tokens(s, s["q"].shape[0])
    n = s["kv_len"][seq] - s["cu_q"].diff()[seq] + i
    cs = s["rope"][n]
    q, k, v = _rotate(s["q"].float(), cs).to(dtype), _rotate(s["k"].float(), cs), s["v"].float()
    at, slot = s["page_table"][seq, n // page], n % page
    if case["bits"] == 16:
        s["cache"][at, :, 0, slot] = k.to(dtype)
        s["cache"][at, :, 1, slot] = v.to(dtype)
        return {"q": q, "cache": s["cache"]}
    kc, vc, kp, vp = _parts(s["cache"], page, dim)
    ck, sk, mk = _quantise(k)
    cv, sv, mv = _quantise(v)
    kc[at, :, slot] = _packed_bytes(ck)
    vc[at, :, slot] = _packed_bytes(cv)
    kp[at, :, slot] = torch.stack([sk, mk], -1)
    vp[at, :, slot] = torch.stack([sv, mv], -1)
    return {"q": q, "k": _values(ck, sk, mk).to(dtype), "v": _values(cv, sv, mv).to(dtype)}


def _cached(case, cache, pages):
    """Keys and values of pages [..., n] in fp32, as [..., n * page, hkv, dim]."""
    page, dim = case["page"], case["dim"]
    data = cache[pages]
    if case["bits"] == 16:
        both = [data[..., i, :, :] for i in (0, 1)]
        both = [x.float() for x in both]
    else:
        kc, vc, kp, vp = _parts(data, page, dim)
        both = [_values(torch.stack([c & 15, c >> 4], -1).flatten(-2).float(), p[..., 0], p[..., 1])
                for c, p in ((kc, kp), (vc, vp))]
    return [x.transpose(-3, -2).flatten(-4, -3) for x in both]


def _plain_paged(s):
    q, cu_q = s["q"], s["cu_q"]
    k, v = _cached(s["case"], s["cache"], s["page_table"])
    o = _attend(s, _padded(q, cu_q, s["new_longest"]), k, v, cu_q.diff(), s["kv_len"], True)
    return o[_tokens(s, q.shape[0])].to(q.dtype)


# ----------------------------------------------------------------------------- work and the exact answer

def _pairs(new, past, causal):
    """Query and key pairs that see each other."""
    if not causal:
        return sum(n * (n + p) for n, p in zip(new, past))
    return sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))


def work(case):
    new, past = _lengths(case)
    rows, total = sum(new), sum(new) + sum(past)
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if case["op"] == "packed":
        return {"bytes": 2 * dim * (2 * rows * hq + 2 * total * hkv), "flops": 4 * dim * hq * _pairs(new, past, case["causal"])}
    held = 4 * dim if case["bits"] == 16 else dim + dim // 4  # bytes of a token's key and value of one head
    if case["op"] == "append":
        out = held + (0 if case["bits"] == 16 else 4 * dim)
        return {"bytes": 2 * dim * rows * (2 * hq + 2 * hkv) + rows * hkv * out + rows * dim * 4,
                "flops": 3 * dim * rows * (hq + hkv)}
    return {"bytes": total * hkv * held + 4 * dim * rows * hq, "flops": 4 * dim * hq * _pairs(new, past, True)}


def _exact_attend(q, k, v, causal, scale):
    """q [Lq, hq, D], k, v [Lk, hkv, D] in 64 bits -> [Lq, hq, D]; a query that sees nothing gives zeros."""
    lq, hq, _ = q.shape
    lk, hkv, _ = k.shape
    out = torch.zeros_like(q)
    for h in range(hq):
        kh = h // (hq // hkv)
        for a in range(0, lq, 4096):
            b = min(lq, a + 4096)
            end = lk - lq + b if causal else lk  # keys that the last of these queries sees
            if end <= 0:
                continue
            score = (q[a:b, h] @ k[:end, kh].T) * scale
            if causal:
                i = torch.arange(a, b, device="cuda")[:, None] + (lk - lq)
                score.masked_fill_(torch.arange(end, device="cuda") > i, -math.inf)
            w = torch.softmax(score, -1)
            out[a:b, h] = torch.where(score.amax(-1, keepdim=True) == -math.inf, 0.0, w @ v[:end, kh])
    return out


def _exact_held(x):
    """What a 4-bit cache holds for rows x in 64 bits."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    least = g.min(-1, keepdim=True).values
    step = ((g.max(-1, keepdim=True).values - least) / 15).bfloat16().double()
    least = least.bfloat16().double()
    codes = ((g - least) / step).round().clamp(0, 15)
    return torch.where(step > 0, least + step * codes, least).reshape(x.shape)


def _exact_rows(case, cache, pages, count):
    """The first `count` keys and values of a sequence with these pages, in 64 bits, [count, hkv, dim]."""
    page, dim, hkv = case["page"], case["dim"], case["hkv"]
    n = torch.arange(count, device="cuda")
    at, slot = pages[n // page].long()[:, None], (n % page)[:, None]
    head = torch.arange(hkv, device="cuda")
    if case["bits"] == 16:
        return cache[at, head, 0, slot].double(), cache[at, head, 1, slot].double()
    both, codes, cache = [], page * dim // 2, cache.flatten(-2)
    for i in (0, 1):
        first = i * codes + slot * (dim // 2)
        raw = cache[at[..., None], head[:, None], first[..., None] + torch.arange(dim // 2, device="cuda")]
        held = torch.stack([raw.remainder(16), raw.div(16, rounding_mode="floor")], -1).reshape(count, hkv, dim).double()
        first = 2 * codes + (i * page + slot) * (dim // GROUP * 4)
        raw = cache[at[..., None], head[:, None], first[..., None] + torch.arange(dim // GROUP * 4, device="cuda")]
        step, least = raw.contiguous().view(torch.bfloat16).double().reshape(count, hkv, dim // GROUP, 2).unbind(-1)
        both.append(held * step.repeat_interleave(GROUP, -1) + least.repeat_interleave(GROUP, -1))
    return both


def exact(case, seed):
    s = prepare(case, seed)
    new, past = _lengths(case)
    at = _starts(new)
    if case["op"] == "packed":
        ends = _starts([n + p for n, p in zip(new, past)])
        return torch.cat([_exact_attend(s["q"][at[b]:at[b + 1]].double(), s["k"][ends[b]:ends[b + 1]].double(),
                                        s["v"][ends[b]:ends[b + 1]].double(), case["causal"], case["dim"] ** -0.5)
                          for b in range(case["batch"])])
    if case["op"] == "paged":
        outs = []
        for b in range(case["batch"]):
            k, v = _exact_rows(case, s["cache"], s["page_table"][b], new[b] + past[b])
            outs.append(_exact_attend(s["q"][at[b]:at[b + 1]].double(), k, v, True, case["dim"] ** -0.5))
        return torch.cat(outs)
    half = case["dim"] // 2
    n = torch.cat([torch.arange(p, p + m, device="cuda") for m, p in zip(new, past)])
    angle = n.double()[:, None] * WAVELENGTH ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotated(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = rotated(s["q"]), rotated(s["k"]), s["v"].double()
    if case["bits"] == 4:
        return {"q": q, "k": _exact_held(k), "v": _exact_held(v)}
    cache = s["cache"].double()
    seq = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), torch.tensor(new, device="cuda"))
    pages, slot = s["page_table"][seq, n // case["page"]].long(), n % case["page"]
    cache[pages, :, 0, slot], cache[pages, :, 1, slot] = k, v
    return {"q": q, "cache": cache}
