"""The choice of tokens at the ends of the logits' and the temperature's ranges, with top_p inside the distribution."""

import pytest
import torch

from smolvla_mujoco_libero_b200 import _lib as L
from tests.test_gpu_answer import FP32, gen, tokens_check

pytestmark = pytest.mark.gpu

TOP_P = [0.3, 0.5, 0.7, 0.9, 0.95, 0.99, 0.999, 1.0]


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(reset=True)
    yield
    torch.cuda.synchronize()
    assert L.device_error(reset=True) == 0


@pytest.mark.parametrize("vocab", [300, 6000])
@pytest.mark.parametrize("spread,temperature", [
    (None, 3e38),                                               # +-3.4e38: differences beyond fp32
    (8e37, 1e38), (1e36, 1e36), (3e30, 1e30),
    (1e-37, 1e-37), (2.0 ** -100, 2.0 ** -101), (1e-20, 2e-20),  # 120 / temperature beyond fp32
    (1e-43, 1e-43),                                             # subnormal logits and temperature
    (1.0, 1e-30), (1e25, 1e-30),                                # only the largest is left
])
def test_top_p_where_differences_or_their_quotients_leave_fp32(vocab, spread, temperature):
    x = torch.randn(8, vocab, generator=gen(vocab)).double()
    most = torch.finfo(FP32).max
    x = torch.where(x > 0, most, -most) if spread is None else (x * spread).clamp(-most, most)
    x = x.float()
    u = torch.rand(8, generator=gen(vocab + 1))
    tokens_check(x, u, temperature=temperature, top_p=TOP_P)
    tokens_check(x, u, temperature=temperature, top_p=TOP_P, top_k=vocab - 7)
    tokens_check(x, u, temperature=temperature, top_p=TOP_P, min_p=0.01)
    x[:, ::3] = -torch.inf
    tokens_check(x, u, temperature=temperature, top_p=TOP_P[::-1])
