"""Plain forms of the serving operators in 64 bits (CPU), one sequence and head at a time, with what the tests derive
their tolerances from.

Attention returns beside the result, per output element, ``spread = sum_j p_j |v_j|`` (what a relative error of the
probabilities or of the values can move) and per row ``size = max_j scale sum_d |q_d| |k_jd|`` (what the rounding of a
score's sum is relative to).  For a 4-bit cache |k| and |v| are |low| + step code, the magnitudes that are added up.
"""

from __future__ import annotations

import math

import torch

GROUP = 32


def attend(q, k, v, seen, scale, k_size=None, v_size=None):
    """q [L, Hq, D], k / v [N, Hkv, D] fp64; seen[i]: query i sees keys 0 .. seen[i] - 1 -> (o, spread, size)."""
    L, hq, _ = q.shape
    g = hq // k.shape[1]
    k_size, v_size = (k.abs() if k_size is None else k_size), (v.abs() if v_size is None else v_size)
    o, spread, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(L, hq, dtype=q.dtype)
    for i in range(L):
        n = seen[i]
        if n <= 0:
            continue
        for h in range(hq):
            kh = h // g
            s = (k[:n, kh] @ q[i, h]) * scale
            p = torch.softmax(s, 0)
            o[i, h] = p @ v[:n, kh]
            spread[i, h] = p @ v_size[:n, kh]
            size[i, h] = (k_size[:n, kh] @ q[i, h].abs()).max() * scale
    return o, spread, size


def attend_dense(q, k, v, seen, scale, k_size=None, v_size=None):
    """The same, a head at a time (longer sequences)."""
    L, hq, _ = q.shape
    g, n = hq // k.shape[1], k.shape[0]
    k_size, v_size = (k.abs() if k_size is None else k_size), (v.abs() if v_size is None else v_size)
    hidden = torch.arange(n)[None] >= torch.as_tensor(seen)[:, None]
    o, spread, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(L, hq, dtype=q.dtype)
    some = ~hidden.all(1)
    for h in range(hq):
        kh = h // g
        s = (q[:, h] @ k[:, kh].T * scale).masked_fill(hidden, -math.inf)
        p = torch.softmax(s[some], -1)
        o[some, h], spread[some, h] = p @ v[:, kh], p @ v_size[:, kh]
        size[some, h] = (q[some, h].abs() @ k_size[:, kh].T * scale).masked_fill(hidden[some], 0).amax(-1)
    return o, spread, size


def causal_seen(n_q: int, n_k: int, causal: bool = True) -> list[int]:
    return [min(max(n_k - n_q + i + 1, 0), n_k) if causal else n_k for i in range(n_q)]


def attention_tolerance(o, spread, size, dtype, dim, weight_unit=None, floor=0.0):
    """Bound of |kernel - o| per element.

    unit: half a step of the output type.  The output is rounded once (unit |o|); the weights of the second product are
    rounded once (weight_unit spread).  The relative error of an fp32 weight is the error of its score: dim products and
    sums, each off by at most 2^-23 (tensor cores may truncate) of the magnitudes, dim + 8 of them with the scale factors,
    in the weight and again in the sum that divides; plus 2^-22 for each of two exponentials and divisions.  floor:
    what weights below the second product's normal range lose.  The second order is covered by 2%, and so is an exponential
    by polynomial (2.6e-6 relative, in the weight and in the sum 5.2e-6; 2% of the smallest weight_unit, 2^-11, is 9.7e-6).
    """
    unit = torch.finfo(dtype).eps / 2
    weight_unit = unit if weight_unit is None else weight_unit
    score = 2 * (dim + 8) * 2.0 ** -23 * size[..., None] + 8 * 2.0 ** -22
    # exp(x) - 1 <= 2 x for the small x here
    return 1.02 * (unit * o.abs() + (weight_unit + 2 * score) * spread) + floor + 1e-30


def rotate(x, cs):
    """Rotate-half in fp32, products and their sum rounded one by one; x [T, H, D] fp32, cs [T, D / 2, 2]."""
    x1, x2 = x.chunk(2, -1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def quantise(x):
    """fp32 [..., D] -> (codes uint8 [..., D], step, low bf16 [..., D / 32])."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((hi - lo) / torch.tensor(15.0)).bfloat16()
    low = lo.bfloat16()
    s = step.float()
    codes = torch.where(s > 0, torch.round((g - low.float()) / s), torch.zeros_like(g)).clamp(0, 15).nan_to_num(0.0)
    return codes.flatten(-2).to(torch.uint8), step.squeeze(-1), low.squeeze(-1)


def held(codes, step, low):
    """What codes stand for, fp32."""
    g = codes.float().unflatten(-1, (-1, GROUP))
    return (g * step.float().unsqueeze(-1) + low.float().unsqueeze(-1)).flatten(-2)


def split4(cache, page, dim):
    """Views of a 4-bit cache [..., page, dim + dim / 4]: key codes, value codes [..., page, dim / 2] and their (step, low) pairs."""
    n, g = page * dim // 2, page * dim // GROUP * 4
    cache = cache.flatten(-2)
    codes = [cache[..., i * n:(i + 1) * n].unflatten(-1, (page, dim // 2)) for i in (0, 1)]
    pairs = [cache[..., 2 * n + i * g:2 * n + (i + 1) * g].view(torch.bfloat16).unflatten(-1, (page, dim // GROUP, 2))
             for i in (0, 1)]
    return codes, pairs


def pack4(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpack4(data):
    return torch.stack([data & 15, data >> 4], -1).flatten(-2)


def entry(cache, page, dim, page_id, slot, which):
    """Key (which 0) or value (1) of an entry, all kv heads, fp32 [Hkv, D]; and its magnitude."""
    if cache.dim() == 5:
        x = cache[page_id, :, which, slot].float()
        return x, x.abs()
    codes, pairs = split4(cache[page_id], page, dim)
    c, p = unpack4(codes[which][:, slot]), pairs[which][:, slot]
    return held(c, p[..., 0], p[..., 1]), held(c, p[..., 0].abs(), p[..., 1].abs())


def rows(cache, page, dim, table, n):
    """The first n entries of a sequence with page table row `table`: (k, v, k_size, v_size) fp64 [n, Hkv, D]."""
    out = [[], [], [], []]
    for i in range(n):
        pid, slot = int(table[i // page]), i % page
        for which in (0, 1):
            x, a = entry(cache, page, dim, pid, slot, which)
            out[which].append(x.double())
            out[2 + which].append(a.double())
    hkv = cache.shape[1]
    return [torch.stack(o) if o else torch.zeros(0, hkv, dim, dtype=torch.float64) for o in out]


def append(cache, page, k, v, cu_q, kv_len, table, cs=None, pos=None, q=None):
    """kv_append on the CPU: changes `cache` in place, returns (q, k, v) with k / v as the cache holds them."""
    dtype, dim = k.dtype, k.shape[2]
    k32, v32 = k.float().clone(), v.float().clone()
    q32 = None if q is None else q.float().clone()
    where = {}
    for b in range(len(cu_q) - 1):
        n_new = int(cu_q[b + 1] - cu_q[b])
        for i in range(n_new):
            where[int(cu_q[b]) + i] = (b, int(kv_len[b]) - n_new + i)
    for t, (b, n) in where.items():
        if cs is not None:
            p = min(max(int(pos[t]) if pos is not None else n, 0), cs.shape[0] - 1)
            k32[t:t + 1] = rotate(k32[t:t + 1], cs[p:p + 1])
            if q is not None:
                q32[t:t + 1] = rotate(q32[t:t + 1], cs[p:p + 1])
    out_k, out_v = k32.to(dtype), v32.to(dtype)
    if cache.dim() == 4:
        parts = [quantise(k32), quantise(v32)]
        out_k, out_v = held(*parts[0]).to(dtype), held(*parts[1]).to(dtype)
    for t, (b, n) in where.items():
        if n < 0 or n // page >= table.shape[1] or not 0 <= int(table[b, n // page]) < cache.shape[0]:
            continue
        pid, slot = int(table[b, n // page]), n % page
        if cache.dim() == 5:
            cache[pid, :, 0, slot], cache[pid, :, 1, slot] = out_k[t], out_v[t]
        else:
            codes, pairs = split4(cache[pid], page, dim)
            for which in (0, 1):
                c, s, m = parts[which]
                codes[which][:, slot] = pack4(c[t])
                pairs[which][:, slot] = torch.stack([s[t], m[t]], -1)
    return None if q is None else q32.to(dtype), out_k, out_v
