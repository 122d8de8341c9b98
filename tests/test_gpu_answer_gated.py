"""Gated products with fp32 outputs: the activation's error does not grow with the gate."""

import pytest
import torch

from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_answer import DEV, FP32, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("impl", [L.LINEAR_FEW, L.LINEAR_MANY], ids=["few", "many"])
@pytest.mark.parametrize("m,k", [(5, 64), (300, 64), (40, 4096)])
@pytest.mark.parametrize("shift", [-7, -10, -13])
def test_gated_products_of_large_gates(impl, m, k, shift):
    """Scales are powers of two and sums below 2^24, so gate and up are exact.  Half steps (2^-24) of the rest: 4 of the exponential
    (2^-22), 1 of its correction, 1 of the sum, 2 of the reciprocal (2^-23), 1 of each product: 10; below 2^-126 the
    sigmoid is 0."""
    n, g = 96, gen(k + m)
    x, w = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, 2 * n))
    xs, ws = torch.full((m,), 2.0 ** shift / (k // 64) ** 0.5), torch.full((2 * n,), 0.125)
    sums = x.double() @ w.double().T
    assert float(sums.abs().max()) < 2 ** 24
    gate, up = (sums * float(xs[0]) * 0.125).chunk(2, -1)
    assert shift < -7 or float(gate.min()) < -90
    got = ops.linear_i8_rows(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), gated=True, dtype=FP32, impl=impl).double().cpu()
    y = gate * torch.sigmoid(gate) * up
    off = (got - y).abs() / (10.1 * 2.0 ** -24 * y.abs() + (gate * up).abs() * 2.0 ** -126 + 1e-37)
    assert float(off.max()) <= 1, float(off.max())


@pytest.mark.parametrize("impl", [L.LINEAR_FEW, L.LINEAR_MANY], ids=["few", "many"])
@pytest.mark.parametrize("dtype", [FP32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [1e3, 1e10, 1e25, 1e34, 1e36])
def test_gates_beyond_the_exponential(impl, dtype, size):
    """Gates from 1e3 to fp32's end, whose activation is the gate itself or 0; beyond that end an infinity, as the product's."""
    m, n, k, g = 7, 64, 16, gen(3)
    x, w = (torch.randint(1, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, 2 * n))
    w[:n:2] *= -1  # every other gate is negative
    xs, ws = torch.ones(m), torch.cat([torch.full((n,), size), torch.full((n,), 1e-3 / size)])
    gate, up = ((x.double() @ w.double().T) * ws.double()).chunk(2, -1)
    finite = gate < torch.finfo(FP32).max
    got = ops.linear_i8_rows(x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), gated=True, dtype=dtype, impl=impl).double().cpu()
    y = torch.where(gate > 0, gate * up, 0.0)
    off = 2.0 ** -24 * 12 + (torch.finfo(dtype).eps / 2 if dtype != FP32 else 0)
    live = finite & (gate > -torch.finfo(FP32).max)
    assert bool(((got - y).abs() <= off * y.abs() + 1e-30)[live].all())
    assert bool((got[~finite] == torch.inf).all())
    assert size > 1e25 or bool(live.all())  # (sums reach 16 127^2 = 2.6e5)
