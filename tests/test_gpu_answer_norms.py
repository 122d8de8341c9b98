"""Norms of quantised rows where fp32 statistics need care: a common offset far above the spread, rows whose squares leave
fp32's range, eps 0."""

import pytest
import torch

from oracle import answer as A
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_answer import BF16, DEV, FP16, dev, gen, rows_check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(reset=True)
    yield
    torch.cuda.synchronize()
    assert L.device_error(reset=True) == 0


def params(k, dtype, seed):
    g = gen(seed)
    return (1 + 0.3 * torch.randn(k, generator=g)).to(dtype), (0.2 * torch.randn(k, generator=g)).to(dtype)


@pytest.mark.parametrize("k", [960, 77, 768, 4097, 20001])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_layernorm_of_constant_rows_is_its_bias(k, dtype):
    w, b = params(k, dtype, k)
    x = torch.tensor([1.0, -3.3, 1000.0, 10000.0, 30000.0, -65000.0, 1e-6]).to(dtype)[:, None].expand(-1, k).contiguous()
    r = torch.tensor([0.1, 0.01, 1e-3, 0.3, 0.7, 5.0, 1e-7]).to(dtype)[:, None].expand(-1, k).contiguous()
    for residual in (None, dev(r)):
        got = ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b), residual=residual)
        scale = b.float().abs().amax() / torch.tensor(127.0)
        assert bool((got.scale.cpu() == scale).all())
        assert bool((got.codes.cpu() == torch.round(b.float() / scale).to(torch.int8)).all())


@pytest.mark.parametrize("k", [960, 77, 4097])
@pytest.mark.parametrize("offset", [30.0, 1000.0, 30000.0])
def test_layernorm_of_rows_far_from_zero(k, offset):
    """x a constant, the residual the spread: fp16 both, their sum in fp32."""
    w, b = params(k, FP16, k)
    x = torch.full((6, k), offset).to(FP16)
    x[3:] *= -1
    r = torch.randn(6, k, generator=gen(k + 1)) * torch.tensor([1.0, 0.1, 10.0, 1.0, 0.1, 10.0])[:, None]
    r = r.to(FP16)
    kw = dict(residual=r, weight=w, bias=b, smooth=None)
    rows_check(x, kw, ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b), residual=dev(r)))


@pytest.mark.parametrize("k", [960, 77, 4097])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_layernorm_of_rows_constant_but_for_one_element(k, dtype):
    """Spreads of a step of the type over sqrt(k), far below the rows' mean; every h exact."""
    w, b = params(k, dtype, k)
    x = torch.tensor([1.0, -3.3, 1000.0, 10000.0, 30000.0, -60000.0]).to(dtype)[:, None].expand(-1, k).contiguous()
    x[:, k // 3] = (x[:, 0].float() * (1 + 2 * torch.finfo(dtype).eps)).to(dtype)
    kw = dict(residual=None, weight=w, bias=b, smooth=None)
    rows_check(x, kw, ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b)))


def test_layernorm_of_rows_beyond_the_squares_range():
    """Means and spreads up to the type's end, k from a few on."""
    for k in (3, 16, 960, 2049):
        w, b = params(k, BF16, k)
        x = torch.randn(7, k, generator=gen(k + 2)) * torch.tensor([1e18, 1e25, 1e30, 1e37, 1e37, 1e20, 1e36])[:, None]
        x = (x + torch.tensor([1e22, 0.0, 3e38, 3e38, -2e38, 1e29, 1e31])[:, None]).clamp(-3.3e38, 3.3e38).to(BF16)
        kw = dict(residual=None, weight=w, bias=b, smooth=None)
        rows_check(x, kw, ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b)))


@pytest.mark.parametrize("k", [960, 77, 4096, 20001])
@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
def test_norms_of_tiny_rows(k, layer):
    """Squares below fp32's range, with eps 0 and with eps as small."""
    w, b = params(k, BF16, k)
    x = torch.randn(8, k, generator=gen(k)) * torch.tensor([1e-12, 1e-18, 1e-21, 1e-23, 1e-30, 1e-36, 1e-38, 1.0])[:, None]
    x = x.to(BF16)
    kw = dict(residual=None, weight=w, bias=b if layer else None, smooth=None)
    for eps in (0.0, 2.0 ** -60, 2.0 ** -90, 2.0 ** -120, 2.0 ** -149):
        got = ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b) if layer else None, eps=eps)
        y, _ = A.rows(x, w, kw["bias"], eps)
        normal = (y.abs().amax(-1) > 1e-30).nonzero().flatten()  # (a scale that is subnormal has fewer bits)
        rows_check(x[normal], kw, ops.QuantizedRows(got.codes.cpu()[normal], got.scale.cpu()[normal], None, None), eps)
        assert bool(torch.isfinite(got.scale).all())


@pytest.mark.parametrize("k", [960, 77, 4096])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 1e-5])
def test_norms_of_rows_of_zeros(k, eps):
    w, b = params(k, BF16, k)
    x = torch.zeros(3, k, dtype=BF16)
    x[1] = -0.0
    got = ops.quantize_rows(dev(x), weight=dev(w), eps=eps, want_values=True)
    assert bool((got.scale == 0).all()) and bool((got.codes == 0).all()) and bool((got.values == 0).all())
    got = ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b), eps=eps)
    scale = b.float().abs().amax() / torch.tensor(127.0)
    assert bool((got.scale.cpu() == scale).all())
    assert bool((got.codes.cpu() == torch.round(b.float() / scale).to(torch.int8)).all())


@pytest.mark.parametrize("k", [960, 77, 4097])
def test_layernorm_of_constant_rows_with_eps_0(k):
    w, b = params(k, BF16, k)
    x = torch.tensor([1.0, -3.3, 30000.0, 3e38, 1e-6, 1e-30, 1e-39])[:, None].to(BF16).expand(-1, k).contiguous()
    got = ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b), eps=0.0)
    scale = b.float().abs().amax() / torch.tensor(127.0)
    assert bool((got.scale.cpu() == scale).all())
    assert bool((got.codes.cpu() == torch.round(b.float() / scale).to(torch.int8)).all())


@pytest.mark.parametrize("k", [960, 77])
def test_norms_of_tiny_rows_far_from_their_spread(k):
    """LayerNorm: means of 1e-15 to 1e-35 with a spread of one step of the type in one element; eps 0 and tiny."""
    w, b = params(k, BF16, k)
    x = torch.tensor([1e-15, 1e-20, 1e-25, -1e-30, 1e-35]).to(BF16)[:, None].expand(-1, k).contiguous()
    x[:, k // 2] = (x[:, 0].float() * (1 + 2.0 ** -6)).to(BF16)
    kw = dict(residual=None, weight=w, bias=b, smooth=None)
    for eps in (0.0, 2.0 ** -149):
        rows_check(x, kw, ops.quantize_rows(dev(x), weight=dev(w), bias=dev(b), eps=eps), eps)
