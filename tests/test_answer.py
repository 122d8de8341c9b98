"""CPU checks of the int8 operators of the text model's answers: what the C ABI and the torch layer refuse before any launch,
the descriptors' layouts, and the 64-bit plain forms that the GPU tests compare with."""

import ctypes
import math

import pytest
import torch

from oracle import answer as A
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_capi import _c_sizeof


@pytest.mark.parametrize("cname,pyname", [("svla_quant_rows_desc", "QuantRowsDesc"), ("svla_linear_i8_desc", "LinearI8Desc"),
                                          ("svla_sample_desc", "SampleDesc")])
def test_struct_layouts(cname, pyname, tmp_path):
    assert ctypes.sizeof(getattr(L, pyname)) == _c_sizeof(cname, tmp_path)


# Addresses that are never read: every case below is refused on the host.
def _quant(**kw):
    d = L.QuantRowsDesc()
    d.x, d.codes, d.scale = 0x100000, 0x200000, 0x300000
    d.x_rs = d.residual_rs = d.codes_rs = d.sum_rs = d.values_rs = 960
    d.m, d.k, d.dtype, d.eps = 4, 960, L.DT_BF16, 1e-5
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _linear(**kw):
    d = L.LinearI8Desc()
    d.x, d.xscale, d.w, d.wscale, d.out = 0x100000, 0x200000, 0x300000, 0x400000, 0x500000
    d.x_rs = d.w_rs = 960
    d.out_rs = d.residual_rs = 320
    d.m, d.n, d.k, d.dtype = 4, 320, 960, L.DT_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _sample(**kw):
    d = L.SampleDesc()
    d.logits, d.u, d.tokens = 0x100000, 0x200000, 0x300000
    d.logits_rs, d.batch, d.vocab, d.dtype = 49280, 4, 49280, L.DT_FLOAT
    d.temperature_value, d.top_p_value = 1.0, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


REFUSED = [
    ("svla_quant_rows", _quant, dict(dtype=L.DT_FLOAT), "dtype"),
    ("svla_quant_rows", _quant, dict(k=0), "1 to 32768"),
    ("svla_quant_rows", _quant, dict(k=32769), "1 to 32768"),
    ("svla_quant_rows", _quant, dict(m=-1), "1 to 32768"),
    ("svla_quant_rows", _quant, dict(eps=-1e-6), "eps"),
    ("svla_quant_rows", _quant, dict(eps=math.nan), "eps"),
    ("svla_quant_rows", _quant, dict(eps=math.inf), "eps"),
    ("svla_quant_rows", _quant, dict(bias=0x600000), "bias without weight"),
    ("svla_quant_rows", _quant, dict(x=None), "x is null"),
    ("svla_quant_rows", _quant, dict(x=0x100001), "x must be aligned"),
    ("svla_quant_rows", _quant, dict(x_rs=959), "x has a row stride"),
    ("svla_quant_rows", _quant, dict(residual=0x600000, residual_rs=8), "residual has a row stride"),
    ("svla_quant_rows", _quant, dict(codes=None), "codes is null"),
    ("svla_quant_rows", _quant, dict(codes_rs=900), "codes has a row stride"),
    ("svla_quant_rows", _quant, dict(scale=None), "scale"),
    ("svla_quant_rows", _quant, dict(scale=0x300002), "scale"),
    ("svla_quant_rows", _quant, dict(sum=0x600001), "sum must be aligned"),
    ("svla_quant_rows", _quant, dict(values=0x600000, values_rs=0), "values has a row stride"),
    ("svla_quant_rows", _quant, dict(smooth=0x600002), "smooth"),
    ("svla_linear_i8", _linear, dict(dtype=L.DT_INT32), "dtype"),
    ("svla_linear_i8", _linear, dict(k=0), "k must be"),
    ("svla_linear_i8", _linear, dict(k=131072, x_rs=131072, w_rs=131072), "k must be"),
    ("svla_linear_i8", _linear, dict(m=-1), "negative"),
    ("svla_linear_i8", _linear, dict(n=-1), "negative"),
    ("svla_linear_i8", _linear, dict(n=0x40000000, out_rs=0x40000000), "2^30"),
    ("svla_linear_i8", _linear, dict(impl=3), "impl"),
    ("svla_linear_i8", _linear, dict(gated=1, bias=0x600000), "gated"),
    ("svla_linear_i8", _linear, dict(gated=1, residual=0x600000), "gated"),
    ("svla_linear_i8", _linear, dict(x=None), "x is null"),
    ("svla_linear_i8", _linear, dict(x=0x100008), "16-byte"),
    ("svla_linear_i8", _linear, dict(w=0x300004), "16-byte"),
    ("svla_linear_i8", _linear, dict(x_rs=968), "16"),
    ("svla_linear_i8", _linear, dict(w_rs=900), "w has a row stride"),
    ("svla_linear_i8", _linear, dict(xscale=None), "scale"),
    ("svla_linear_i8", _linear, dict(wscale=0x400002), "scale"),
    ("svla_linear_i8", _linear, dict(bias=0x600001), "bias"),
    ("svla_linear_i8", _linear, dict(out=None), "out is null"),
    ("svla_linear_i8", _linear, dict(out_rs=300), "out has a row stride"),
    ("svla_linear_i8", _linear, dict(out=0x500001), "out must be aligned"),
    ("svla_linear_i8", _linear, dict(residual=0x600000, residual_rs=8), "residual has a row stride"),
    ("svla_sample_tokens", _sample, dict(dtype=L.DT_INT32), "dtype"),
    ("svla_sample_tokens", _sample, dict(vocab=0), "vocab"),
    ("svla_sample_tokens", _sample, dict(vocab=262145, logits_rs=262145), "vocab"),
    ("svla_sample_tokens", _sample, dict(batch=-1), "batch"),
    ("svla_sample_tokens", _sample, dict(temperature_value=-0.5), "temperature"),
    ("svla_sample_tokens", _sample, dict(temperature_value=math.inf), "temperature"),
    ("svla_sample_tokens", _sample, dict(temperature_value=math.nan), "temperature"),
    ("svla_sample_tokens", _sample, dict(top_p_value=-0.1), "top_p"),
    ("svla_sample_tokens", _sample, dict(top_p_value=math.nan), "top_p"),
    ("svla_sample_tokens", _sample, dict(min_p_value=-0.1), "min_p"),
    ("svla_sample_tokens", _sample, dict(logits=None), "logits is null"),
    ("svla_sample_tokens", _sample, dict(logits=0x100002), "logits must be aligned"),
    ("svla_sample_tokens", _sample, dict(logits_rs=49279), "logits has a row stride"),
    ("svla_sample_tokens", _sample, dict(u=None), "u or tokens"),
    ("svla_sample_tokens", _sample, dict(tokens=None), "u or tokens"),
    ("svla_sample_tokens", _sample, dict(top_k=0x600002), "aligned"),
]


@pytest.mark.parametrize("name,make,change,word", REFUSED)
def test_refused_before_any_launch(name, make, change, word):
    lib = L.lib()
    assert getattr(lib, name)(ctypes.byref(make(**change)), None) == 1
    assert word in lib.svla_last_error().decode(), lib.svla_last_error()


@pytest.mark.parametrize("name", ["svla_quant_rows", "svla_linear_i8", "svla_sample_tokens"])
def test_null_descriptors_are_refused(name):
    assert getattr(L.lib(), name)(None, None) == 1


@pytest.mark.parametrize("name,make,change", [("svla_quant_rows", _quant, dict(m=0, x=None)), ("svla_linear_i8", _linear, dict(m=0, x=None)),
                                              ("svla_linear_i8", _linear, dict(n=0, w=None)),
                                              ("svla_sample_tokens", _sample, dict(batch=0, logits=None))])
def test_empty_calls_do_nothing(name, make, change):
    assert getattr(L.lib(), name)(ctypes.byref(make(**change)), None) == 0


@pytest.mark.parametrize("call", [
    lambda: ops.quantize_rows(torch.zeros(2, 8, dtype=torch.bfloat16)),
    lambda: ops.linear_i8_rows(torch.zeros(2, 16, dtype=torch.int8), torch.ones(2), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)),
    lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(ValueError, match="CUDA tensor"):
        call()


# ----------------------------------------------------------------------------- the oracle against other definitions

def test_oracle_rows():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 40, generator=g).bfloat16()
    w, b = torch.randn(40, generator=g).bfloat16(), torch.randn(40, generator=g).bfloat16()
    y, scale = A.rows(x, weight=w, bias=b, eps=1e-5)
    ref = torch.nn.functional.layer_norm(x.double(), (40,), w.double(), b.double(), 1e-5)
    assert torch.allclose(y, ref, atol=1e-12) and torch.allclose(scale, ref.abs().amax(-1) / 127)
    y, _ = A.rows(x, weight=w, eps=1e-5, residual=x, smooth=torch.full((40,), 2.0))
    assert torch.allclose(y, torch.nn.functional.rms_norm(2 * x.double(), (40,), w.double(), 1e-5) / 2, atol=1e-12)


def test_oracle_product():
    g = torch.Generator().manual_seed(1)
    x, w = (torch.randint(-127, 128, (n, 30), generator=g, dtype=torch.int8) for n in (4, 6))
    xs, ws = torch.rand(4, generator=g), torch.rand(6, generator=g) / 1000
    deq = (x.double() * xs.double()[:, None]) @ (w.double() * ws.double()[:, None]).T
    assert torch.allclose(A.product(x, xs, w, ws)[0], deq)
    gate, up = deq.chunk(2, -1)
    assert torch.allclose(A.product(x, xs, w, ws, gated=True)[0], torch.nn.functional.silu(gate) * up)


def test_oracle_tokens_follow_the_distribution():
    """Over a grid of random numbers each kept token comes up as often as its share says, in the order of the indices."""
    x = torch.tensor([0.0, 2.0, 1.0, 2.0, -1.0, 0.5])
    p = torch.softmax(x.double() / 0.8, -1)
    n = 4000
    drawn = [A.sample(x, (i + 0.5) / n, temperature=0.8)[0] for i in range(n)]
    assert drawn == sorted(drawn)
    for i in range(6):
        assert abs(drawn.count(i) / n - float(p[i])) <= 1.0 / n
    assert {A.sample(x, (i + 0.5) / 50, top_k=3)[0] for i in range(50)} == {1, 2, 3}
    assert {A.sample(x, (i + 0.5) / 50, top_k=1)[0] for i in range(50)} == {1}
    assert A.sample(x, 0.3, temperature=0.0)[0] == 1
    # probabilities of the logits 2, 2, 1, 0.5, 0, -1: 0.33, 0.33, 0.12, ... of the rest
    assert {A.sample(x, (i + 0.5) / 50, top_p=0.5)[0] for i in range(50)} == {1, 3}
    assert {A.sample(x, (i + 0.5) / 50, min_p=0.3)[0] for i in range(50)} == {1, 2, 3}
    assert A.sample(torch.full((4,), -math.inf), 0.5)[0] == -1
