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
