"""Quantised rows, int8 products of them and the choice of tokens on the GPU, against plain forms in 64 bits
(oracle/answer.py, which derives the bars).  Rows without a norm and the tokens themselves: equal."""

import itertools
import math

import pytest
import torch

from oracle import answer as A
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(reset=True)
    yield
    torch.cuda.synchronize()
    assert L.device_error(reset=True) == 0


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(x):
    return None if x is None else x.to(DEV)


# ----------------------------------------------------------------------------- quantised rows

def row_inputs(m, k, dtype, norm="none", residual=False, smooth=False, seed=0):
    g = gen(seed)
    x = torch.randn(m, k, generator=g)
    x[:, k // 5::k // 4 + 1] *= 8
    kw = {"residual": (2 * torch.randn(m, k, generator=g)).to(dtype) if residual else None,
          "weight": (1 + 0.3 * torch.randn(k, generator=g)).to(dtype) if norm != "none" else None,
          "bias": (0.2 * torch.randn(k, generator=g)).to(dtype) if norm == "layer" else None,
          "smooth": torch.exp(0.5 * torch.randn(k, generator=g)) if smooth else None}
    return x.to(dtype), kw


def rows_check(x, kw, got, eps=1e-5):
    """codes, scale, sum and values against the definition."""
    y, scale = A.rows(x, eps=eps, **kw)
    rel, off = A.rows_tolerance(x, eps=eps, **kw)
    codes, gs = got.codes.cpu(), got.scale.cpu()
    assert bool(((gs.double() - scale).abs() <= rel * scale + 1e-44).all()), float(((gs - scale).abs() / scale).max())
    live = scale > 0
    q = y[live] / scale[live, None]
    assert bool(((codes[live].double() - q).abs() <= 0.5 + off[live, None]).all())
    assert bool((codes[~live] == 0).all()) and int(codes.abs().max()) <= 127
    if kw["residual"] is not None:
        assert torch.equal(got.sum.cpu(), (x.float() + kw["residual"].float()).to(x.dtype))
    if got.values is not None:
        assert torch.equal(got.values.cpu(), (codes.float() * gs[:, None]).to(x.dtype))


SHAPES = [(1, 960), (3, 2560), (1300, 960), (7, 1), (5, 7), (2, 16), (1, 1023), (9, 1024), (1200, 1024), (3, 1025), (4, 4096),
          (2, 4097), (2, 8192), (1, 11008), (2, 16384), (1, 32768), (1, 20001), (1185, 24)]


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows(shape, norm, dtype):
    for residual, smooth in itertools.product([False, True], repeat=2):
        x, kw = row_inputs(*shape, dtype, norm, residual, smooth, seed=shape[1])
        got = ops.quantize_rows(dev(x), **{n: dev(t) for n, t in kw.items()}, want_values=smooth)
        assert (got.sum is not None) == residual and (got.values is not None) == smooth
        rows_check(x, kw, got)


@pytest.mark.parametrize("shape", [(1, 960), (1300, 960), (40, 2560), (3, 77), (2, 16384)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_rows_without_a_norm_are_exact(shape, dtype):
    """fp32 sum, IEEE quotients: the codes of the definition bit for bit, halves among them."""
    x, kw = row_inputs(*shape, dtype, residual=True, seed=5)
    x[0] = 0
    x[0, 0], kw["residual"][0] = 127, 0
    x[0, 1:7] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 63.5]).to(dtype)  # scale 1: ties to even
    h = x.float() + kw["residual"].float()
    scale = h.abs().amax(-1) / torch.tensor(127.0)
    got = ops.quantize_rows(dev(x), residual=dev(kw["residual"]))
    assert torch.equal(got.scale.cpu(), scale)
    assert torch.equal(got.codes.cpu(), torch.round(h / scale[:, None]).to(torch.int8))


def test_rows_strided_and_in_place():
    x, kw = row_inputs(50, 960, BF16, "rms", residual=True, seed=6)
    wide, res = torch.full((50, 1000), 7.0, dtype=BF16, device=DEV), dev(kw["residual"]).clone()
    wide[:, 8:968] = dev(x)
    codes = torch.full((50, 976), 99, dtype=torch.int8, device=DEV)
    got = ops.quantize_rows(wide[:, 8:968], weight=dev(kw["weight"]), residual=res, sum=res, codes=codes[:, :960])
    rows_check(x, kw, got)
    assert got.sum is res and bool((codes[:, 960:] == 99).all()) and bool((wide[:, :8] == 7).all())
    # one element off: no 16-byte loads
    wide[:, 9:969] = dev(x)
    again = ops.quantize_rows(wide[:, 9:969], weight=dev(kw["weight"]), residual=dev(kw["residual"]), sum=wide[:, 9:969])
    assert torch.equal(again.codes, got.codes) and torch.equal(wide[:, 9:969], res)
    rows_check(x, kw, again)


@pytest.mark.parametrize("k", [960, 4096, 77])
def test_rows_of_zeros_infinities_and_extremes(k):
    g = gen(9)
    x = torch.randn(8, k, generator=g).to(BF16)
    x[0] = 0
    x[1, 3], x[2, 5], x[3, k - 1] = math.inf, math.nan, -math.inf
    x[4] *= 1e-38
    x[5] = (x[5].float() * 1e38).clamp(-3e38, 3e38).to(BF16)
    x[6] = 0
    x[6, k // 2] = 3e38
    got = ops.quantize_rows(dev(x), want_values=True)
    scale, codes = got.scale.cpu(), got.codes.cpu()
    assert scale[0] == 0 and bool((codes[0] == 0).all()) and bool((got.values[0] == 0).all())
    assert bool(torch.isnan(scale[1:4]).all()) and bool((codes[1:4] == 0).all()) and bool(torch.isnan(got.values[1:4]).all())
    keep = [4, 5, 6, 7]
    rows_check(x[keep], dict(residual=None, weight=None, bias=None, smooth=None),
               ops.QuantizedRows(codes[keep], scale[keep], None, got.values[keep]))
    # norms of rows whose squares leave fp32's range, and of a row of zeros
    w, b = torch.ones(k, dtype=BF16), torch.zeros(k, dtype=BF16)
    for kw in (dict(weight=w, bias=None), dict(weight=w, bias=b)):
        got = ops.quantize_rows(dev(x), **{n: dev(t) for n, t in kw.items()})
        assert bool(torch.isnan(got.scale[1:4]).all()) and got.scale[0] == 0
        keep = [0, 5, 6, 7]
        rows_check(x[keep], dict(residual=None, smooth=None, **kw), ops.QuantizedRows(got.codes[keep], got.scale[keep], None, None))


# ----------------------------------------------------------------------------- products

def product_inputs(m, n, k, gated=False, seed=0):
    g = gen(seed)

    def codes(rows):
        x = torch.full((rows, -(-k // 16) * 16), 111, dtype=torch.int8)  # what stands behind k counts for nothing
        x[:, :k] = torch.randint(-127, 128, (rows, k), generator=g, dtype=torch.int8)
        return x[:, :k]
    rows = 2 * n if gated else n
    size = 1 / (73 * math.sqrt(k))
    return codes(m), torch.rand(m, generator=g) + 0.1, codes(rows), (torch.rand(rows, generator=g) + 0.1) * size


def product_check(m, n, k, dtype, gated=False, bias=False, residual=False, seed=0, impl=L.LINEAR_AUTO):
    x, xs, w, ws = product_inputs(m, n, k, gated, seed)
    g = gen(seed + 1)
    b = torch.randn(n, generator=g) if bias else None
    r = torch.randn(m, n, generator=g).to(dtype) if residual else None
    y, size = A.product(x, xs, w, ws, b, r, gated)
    pad = lambda t: torch.nn.functional.pad(t, (0, -t.shape[1] % 16), value=111).to(DEV)[:, :t.shape[1]]  # noqa: E731
    out = torch.full((m, n + 5), 9.0, dtype=dtype, device=DEV)
    # rows a multiple of 16 bytes apart, whatever n is; the residual likewise
    wide = torch.full((m + 1, -(-n // 16) * 16 + 16), 9.0, dtype=dtype, device=DEV)
    res = None if r is None else torch.full_like(wide, 5.0)
    if r is not None:
        res[:m, :n] = dev(r)
    for o in (None, out[:, :n], wide[:m, :n]):
        given = res[:m, :n] if r is not None and o is not None and o.stride(0) == wide.stride(0) else dev(r)
        got = ops.linear_i8_rows(pad(x), dev(xs), pad(w), dev(ws), dev(b), given, gated, dtype, o, impl)
        assert got.dtype == dtype and got.shape == (m, n)
        off = (got.double().cpu() - y).abs() / A.product_tolerance(y, size, dtype)
        assert float(off.max()) <= 1, float(off.max())
    assert bool((out[:, n:] == 9).all()) and bool((wide[:m, n:] == 9).all()) and bool((wide[m:] == 9).all())
    if r is not None:  # in place
        got = ops.linear_i8_rows(pad(x), dev(xs), pad(w), dev(ws), dev(b), res[:m, :n], gated, dtype, res[:m, :n], impl)
        assert torch.equal(got, wide[:m, :n]) and bool((res[:m, n:] == 5).all()) and bool((res[m:] == 5).all())


FEW = [(1, 1600, 960), (1, 1, 1), (1, 7, 3), (2, 130, 77), (16, 128, 128), (17, 960, 2560), (33, 100, 16), (64, 4096, 960), (65, 129, 129),
       (128, 320, 4096), (129, 257, 640), (200, 960, 960), (256, 1000, 144)]
MANY = [(1, 1, 1), (257, 256, 128), (300, 1000, 960), (700, 328, 200), (512, 129, 77), (1000, 2560, 960), (11, 500, 2000), (2500, 8, 16)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", FEW, ids=str)
def test_product_of_few_rows(shape, dtype):
    product_check(*shape, dtype, seed=shape[1], impl=L.LINEAR_FEW)
    product_check(*shape, dtype, bias=True, residual=True, seed=shape[1], impl=L.LINEAR_FEW)
    product_check(*shape, dtype, gated=True, seed=shape[1], impl=L.LINEAR_FEW)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_product_of_many_rows(shape, dtype):
    product_check(*shape, dtype, seed=shape[1], impl=L.LINEAR_MANY)
    product_check(*shape, dtype, bias=True, residual=True, seed=shape[1], impl=L.LINEAR_MANY)
    product_check(*shape, dtype, gated=True, seed=shape[1], impl=L.LINEAR_MANY)


# ----------------------------------------------------------------------------- tokens

def tokens_check(logits, u, **kw):
    """Every row against the definition; kw: lists with a value per row, or numbers."""
    args = {n: (torch.tensor(v, dtype=torch.int32 if n == "top_k" else FP32).to(DEV) if isinstance(v, list) else v) for n, v in kw.items()}
    token, logprob = ops.sample_tokens(logits.to(DEV), u.to(DEV), **args)
    token, logprob = token.cpu().tolist(), logprob.cpu().tolist()
    for b in range(len(u)):
        one = {n: v[b] if isinstance(v, list) else v for n, v in kw.items()}
        want, lp, _ = A.sample(logits[b], float(u[b]), **one)
        assert token[b] == want, (b, token[b], want, one)
        assert (math.isnan(lp) and math.isnan(logprob[b])) or abs(logprob[b] - lp) <= 2.0 ** -24 * abs(lp) + 1e-12, (b, logprob[b], lp)


def logits_of(batch, vocab, dtype, spread=2.5, seed=0):
    g = gen(seed)
    x = torch.randn(batch, vocab, generator=g) * spread
    return x.to(dtype), torch.rand(batch, generator=g)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 5, 31, 256, 1000, 1025, 2049, 4097, 9000])
def test_tokens(vocab, dtype):
    x, u = logits_of(12, vocab, dtype, seed=vocab)
    tokens_check(x, u)
    tokens_check(x, u, temperature=0.5, top_k=50)
    tokens_check(x, u, top_p=0.9)
    tokens_check(x, u, temperature=1.7, min_p=0.05)
    tokens_check(x, u, temperature=[0.0, 0.1, 0.7, 1.0, 2.0, 5.0, 50.0, 1e6, 1e-6, 1.0, 1.0, 1.0],
                 top_k=[5, 0, -1, 1, 2, 3, 40, 300, 100000, 700, 7, 20], top_p=[1.0, 0.9, 0.5, 0.99, 1.5, 0.0, 0.7, 0.3, 0.6, 0.95, 1.0, 0.8],
                 min_p=[0.0, 0.0, 0.1, 0.0, 0.01, 0.5, 0.0, 0.2, 0.0, 0.0, 1.0, 2.0])


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_tokens_of_a_whole_vocabulary(dtype):
    x, u = logits_of(6, 49280, dtype, seed=3)
    tokens_check(x, u, temperature=[1.0, 0.7, 1.3, 1.0, 0.9, 30.0], top_k=[0, 50, 0, 3000, 20000, 0], top_p=[1.0, 0.95, 0.9, 0.999, 0.5, 0.7],
                 min_p=[0.0, 0.0, 0.0, 0.0, 1e-4, 0.0])


def test_tokens_of_the_largest_vocabulary():
    x, u = logits_of(2, 262144, FP32, spread=1.0, seed=4)
    tokens_check(x, u, top_p=[1.0, 0.97], top_k=[0, 200000])
    tokens_check(torch.zeros(2, 262144, dtype=BF16), torch.tensor([0.25, 0.999]), top_p=[0.5, 1.0], top_k=[0, 777])


@pytest.mark.parametrize("vocab", [600, 5000, 30000])
def test_tokens_with_equal_logits(vocab):
    """All logits equal, and a few levels only: cuts fall among equal logits, more of them than one CTA ranks."""
    u = torch.tensor([0.0, 0.1, 0.5, 0.77, 0.999, 1.0])
    flat = torch.full((6, vocab), -3.0)
    steps = torch.arange(vocab).remainder(3).float().expand(6, vocab).contiguous()
    for x in (flat, steps, steps.to(BF16), -steps):
        tokens_check(x, u)
        tokens_check(x, u, top_k=[1, 2, vocab // 3, vocab // 3 + 1, vocab // 2, vocab - 1])
        tokens_check(x, u, top_p=[0.1, 0.25, 0.5, 0.75, 0.9, 0.01])
        tokens_check(x, u, top_p=0.6, top_k=vocab // 2 + 3, min_p=0.05)


def test_tokens_close_together():
    """Logits a step of fp32 apart: thousands in one bin of the histogram."""
    x = (1.0 + torch.arange(20000).double() * 2.0 ** -23).float().flip(0).expand(4, 20000).contiguous()
    tokens_check(x, torch.tensor([0.1, 0.4, 0.6, 0.9]), top_k=[3, 600, 5000, 19999], top_p=[1.0, 0.5, 0.25, 0.9])
    y = torch.cat([x, torch.full((4, 3000), 40.0)], 1)  # and a plateau above them
    tokens_check(y, torch.tensor([0.1, 0.4, 0.6, 0.9]), top_k=[3100, 10, 0, 2999], top_p=[0.999, 0.5, 0.25, 0.9])


@pytest.mark.parametrize("vocab", [100, 10000])
def test_tokens_of_masked_rows(vocab):
    x, u = logits_of(8, vocab, FP32, seed=11)
    low = torch.finfo(FP32).min
    x[0, 5:] = -math.inf
    x[1, :] = -math.inf
    x[2, 1:] = low
    x[3, 7] = math.nan
    x[4, 9] = math.inf
    x[5] = low
    x[6, ::2] = low
    x[7, :-1] = -math.inf
    for kw in ({}, {"top_k": 10}, {"top_p": 0.8}, {"min_p": 0.3}, {"temperature": 0.0}, {"top_k": 20, "top_p": 0.7, "temperature": 0.6}):
        tokens_check(x, u, **kw)
    tokens_check(torch.full((1, vocab), -0.0).index_fill(1, torch.tensor([vocab // 2]), 0.0), u[:1], temperature=0.0)


def test_settings_that_are_none_give_no_token():
    x, _ = logits_of(9, 50, FP32, seed=12)
    nan = math.nan
    tokens_check(x, torch.tensor([0.5, 0.5, 0.5, 0.5, 0.5, -0.1, 1.1, nan, 0.5]), temperature=[-1.0, nan, math.inf, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0],
                 top_p=[1.0, 1.0, 1.0, -0.1, nan, 1.0, 1.0, 1.0, 1.0], min_p=[0.0] * 8 + [nan])
