"""The serving operators on the GPU where a masked, hidden, huge or missing entry could reach a row that must not know of
it: values at the types' limits, scores of -infinity, groups of very different size, pages that are not there.

Bars as in test_gpu_serving.py (oracle.serving.attention_tolerance), with the floors derived beside each test.
"""

import math

import pytest
import torch

from oracle import serving as S
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_serving import (BF16, DEV, FP16, KERNELS, _no_device_error, filled_cache, gen, ints,  # noqa: F401
                                    packed_inputs, packed_reference, starts, within)

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


@pytest.mark.parametrize("impl", KERNELS)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(3, 1, 64), (4, 2, 128)], ids=str)
@pytest.mark.parametrize("gone", [1, 20, 150])
def test_packed_attention_scores_of_minus_infinity(impl, heads, dtype, gone):
    """The first `gone` keys' scores are -infinity: rows that see no other key give zeros, the others what the keys behind
    give."""
    hq, hkv, d, n = *heads, 200
    q, kv = packed_inputs([n], [n], hq, hkv, d, dtype, seed=41)
    q[..., 5] = q[..., 5].abs() + 0.5
    some, tail = torch.arange(n) >= gone, kv[gone:]
    o, spread, size = packed_reference(q, tail, [n], [n - gone], True)
    kv[:gone, :hkv, 5] = -math.inf
    kvd = kv.to(DEV)
    got = ops.packed_attention(q.to(DEV), kvd[:, :hkv], kvd[:, hkv:], ints([0, n]).to(DEV), impl=impl)
    assert bool((got[:gone] == 0).all())
    within(got[some.to(DEV)], o[some], S.attention_tolerance(o, spread, size, dtype, d)[some])


@pytest.mark.parametrize("heads", [(3, 1, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("gone,total,width", [(2, 5, None), (40, 45, None), (1500, 2000, 200), (2000, 2003, 200)])
def test_paged_attention_scores_of_minus_infinity(heads, gone, total, width):
    """16 bits, the first `gone` entries' scores are -infinity: what rows see behind them, or zeros."""
    hq, hkv, d = heads
    new, page = 5, 16
    cache, table = filled_cache([total], heads, 16, page, BF16, seed=55, width=width)
    q = torch.randn(new, hq, d, generator=gen(56)).to(BF16)
    q[..., 5] = q[..., 5].abs() + 0.5
    k, v = S.rows(cache, page, d, table[0], total)[:2]
    o, spread, size = S.attend_dense(q.double(), k[gone:], v[gone:], S.causal_seen(new, total - gone), d ** -0.5)
    for n in range(gone):
        cache[int(table[0, n // page]), :, 0, n % page, 5] = -math.inf
    got = ops.paged_attention(q.to(DEV), cache.to(DEV), ints([0, new]).to(DEV), ints([total]).to(DEV), table.to(DEV))
    none = [i for i in range(new) if total - new + i < gone]
    assert bool((got[none] == 0).all())
    within(got, o, S.attention_tolerance(o, spread, size, BF16, d))
