"""The serving operators on the GPU where a masked, hidden, huge or missing entry could reach a row that must not know of
it: values at the types' limits, scores of -infinity, groups of very different size, pages that are not there.

Bars as in test_gpu_serving.py (oracle.serving.attention_tolerance), with the floors derived beside each test.
"""

import pytest
import torch

from oracle import serving as S
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_serving import (BF16, DEV, FP16, KERNELS, _no_device_error, ints, packed_inputs,  # noqa: F401
                                    packed_reference, starts, within)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- packed prompts

# every place of a key that the exponentials of a tile treat alike, and the tiles' borders
PLACES = list(range(0, 20)) + [32, 33, 63, 64, 80, 113, 127, 128, 129, 144]


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128)], ids=str)
def test_packed_attention_hidden_values_at_the_limit_of_the_type(impl, heads, dtype):
    """One sequence per place of a value of the type's largest size: rows before it are as if it were not there."""
    hq, hkv, d, n = *heads, 145
    lens = [n] * len(PLACES)
    q, kv = packed_inputs(lens, lens, hq, hkv, d, dtype, seed=40)
    o, spread, size = packed_reference(q, kv, lens, lens, True)
    for i, j in enumerate(PLACES):
        kv[i * n + j, hkv:] = torch.finfo(dtype).max * (-1) ** i
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints(starts(lens)).to(DEV), impl=impl)
    tol = S.attention_tolerance(o, spread, size, dtype, d)
    for i, j in enumerate(PLACES):
        within(got[i * n:i * n + j], o[i * n:i * n + j], tol[i * n:i * n + j], f"place {j}")
