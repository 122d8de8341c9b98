"""Plain forms, in 64 bits on the CPU, of the operators that answer with the text model in int8: quantised rows, products of
such rows, the choice of a token; and what the tests derive their tolerances from."""

from __future__ import annotations

import math

import torch


def rows(x, weight=None, bias=None, eps=1e-5, residual=None, smooth=None):
    """(y, scale) in 64 bits of x [m, k]: codes are y / scale, rounded."""
    h = x.double() + (residual.double() if residual is not None else 0)
    y = h
    if weight is not None:
        d = h - h.mean(-1, keepdim=True) if bias is not None else h
        y = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * weight.double()
        if bias is not None:
            y = y + bias.double()
    if smooth is not None:
        y = y / smooth.double()
    return y, y.abs().amax(-1) / 127


def rows_tolerance(x, weight=None, bias=None, eps=1e-5, residual=None, smooth=None):
    """(relative error of the scale, error of y / scale) that fp32 arithmetic may have.

    A thread adds up at most 32 values, 5 rounds of shuffles join 32 threads and 31 additions as many warps: a statistic is off
    by at most 70 half steps (2^-24) of its magnitudes' sum, its root by half of that.  Beside it: the sum h, the square, the
    reciprocal root (2), the two products with it, the bias' sum, the quotient with smooth, the scale: 10 half steps.  LayerNorm's mean
    is off by 72 half steps of mean |h|, e, which counts against the centred values: relative to the largest y it is 72 (mean |h| / std)
    times the largest weight.  Where the mean is more than 4 deviations the mean of the centred values is taken off as well: it is
    off by 72 half steps of their mean size (at most e above that of the exact ones), both centrings round, and a sum h
    that was rounded is off by half a step of it."""
    half = 2.0 ** -24
    y, scale = rows(x, weight, bias, eps, residual, smooth)
    rel = torch.full_like(scale, (10 + (35 if weight is not None else 0)) * half)
    if bias is not None:
        h = x.double() + (residual.double() if residual is not None else 0)
        d = h - h.mean(-1, keepdim=True)
        e = 72 * half * h.abs().mean(-1)
        again = half * (72 * (d.abs().mean(-1) + e) + d.abs().amax(-1) + e + (2 * h.abs().amax(-1) if residual is not None else 0))
        far = h.mean(-1).square() > 17 * d.square().mean(-1)
        off = torch.where(far, again, e) / torch.sqrt(d.square().mean(-1) + eps)
        w = weight.double().abs() / (smooth.double() if smooth is not None else 1)
        b = bias.double().abs() / (smooth.double() if smooth is not None else 1)
        # the bias may cancel most of a product: errors are relative to the parts
        parts = ((d.abs() / torch.sqrt(d.square().mean(-1, keepdim=True) + eps) * w + b).amax(-1)) / (scale * 127).clamp_min(1e-300)
        rel = rel * parts + off * w.amax() / (scale * 127).clamp_min(1e-300)
    # y / scale is at most 127: y's error, the scale's and the quotient's
    return rel, 127 * (2 * rel + 2 * half)


def product(x, xscale, w, wscale, bias=None, residual=None, gated=False):
    """(y, size) in 64 bits; size bounds what errors are relative to (see product_tolerance)."""
    p = (x.double() @ w.double().T) * xscale.double()[:, None] * wscale.double()
    if gated:
        g, u = p.chunk(2, -1)
        y = g * torch.sigmoid(g) * u
        return y, y.abs() * (2.0 ** 3 + 16 + 5 * g.abs()) + (g * u).abs() * 2.0 ** -102
    size = 3 * p.abs()
    for extra in (bias, residual):
        if extra is not None:
            p = p + extra.double()
            size = size + p.abs()
    return p, size


def product_tolerance(y, size, dtype):
    """fp32's half steps times `size` (3 of the scaled product: the sum's conversion and two scales; one of each later sum; gated:
    2^-21 for the hardware's exponential and reciprocal, 8 half steps, 5 |gate| of the exponent's argument, and as much again for
    the up projection; the hardware's reciprocal gives 0 for what is below 2^-126, gates under -87, so the sigmoid is off by up to
    2^-126 and the product by 2^-126 = 2^-24 2^-102 times |gate up|), and half a step of the output's type."""
    unit = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    return 1.01 * (unit * y.abs() + 2.0 ** -24 * size) + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


UNIT = 2 ** 44


def weights(logits, temperature):
    """Whole-number weights of a row (int64)."""
    x = logits.double()
    return torch.floor(torch.exp((x - x.max()) / temperature) * UNIT + 0.5).long()


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob, kept indices) of one row, walking down the order of logits; token -1 where the row or a setting is none."""
    x = logits.double()
    f = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731  settings are fp32
    u, temperature, top_p, min_p = f(u), f(temperature), f(top_p), f(min_p)
    fine = (not bool(torch.isnan(x).any()) and math.isfinite(float(x.max())) and temperature >= 0 and math.isfinite(temperature) and top_p >= 0
            and min_p >= 0 and 0 <= u <= 1)
    if not fine:
        return -1, math.nan, []
    order = sorted(range(len(x)), key=lambda i: (-float(x[i]), i))
    if temperature == 0:
        return order[0], 0.0, order[:1]
    w = weights(logits, temperature).tolist()
    kept = order[:top_k] if top_k > 0 else order
    kept = [i for n, i in enumerate(kept) if n == 0 or float(w[i]) >= min_p * UNIT]
    if top_p < 1:
        limit, before, some = math.ceil(top_p * float(sum(w[i] for i in kept))), 0, []
        for n, i in enumerate(kept):
            if n and before >= limit:
                break
            some.append(i)
            before += w[i]
        kept = some
    total = sum(w[i] for i in kept)
    target = min(int(u * float(total)), total - 1)
    running = 0
    for i in sorted(kept):
        running += w[i]
        if running > target:
            return i, math.log(w[i] / total), kept
    raise AssertionError
