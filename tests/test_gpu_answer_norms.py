"""Norms of quantised rows where fp32 statistics need care: a common offset far above the spread."""

import pytest
import torch

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
