"""Quantised rows at odd addresses and widths, with what stands around them, and at the ends of what their norms take."""

import pytest
import torch

from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
from tests.test_gpu_answer import BF16, DEV, FP16, dev, row_inputs, rows_check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    L.device_error(reset=True)
    yield
    torch.cuda.synchronize()
    assert L.device_error(reset=True) == 0


def around(x, gap, first):
    """x's rows in one buffer, `gap` elements of 7 between them and `first` before the first and behind the last: (buffer, rows)."""
    m, k = x.shape
    buffer = torch.full((2 * first + m * (k + gap),), 7.0, dtype=x.dtype, device=DEV)
    rows = torch.as_strided(buffer, (m, k), (k + gap, 1), first)
    rows.copy_(x)
    return buffer, rows


def untouched(buffer, rows):
    rest = buffer.clone()
    torch.as_strided(rest, rows.shape, rows.stride(), rows.storage_offset()).fill_(7.0)
    return bool((rest == 7).all())


# widths that leave a warp of the block without any element, others around them
@pytest.mark.parametrize("k", [256, 768, 1280, 1792, 16640, 17152, 255, 257, 512, 960, 2049])
@pytest.mark.parametrize("gap,first", [(0, 1), (1, 1), (1, 2), (4, 3)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_rows_leave_what_is_around_them(k, gap, first, dtype):
    m = 5
    x, kw = row_inputs(m, k, dtype, "rms", residual=True, seed=k)
    x[2, 3] = float("nan")  # values NaN
    keep = torch.tensor([0, 1, 3, 4])
    given = {n: dev(t) for n, t in kw.items()}
    want = ops.quantize_rows(dev(x), **given, want_values=True)  # (16-byte rows where k is a multiple of 8)
    rows_check(x[keep], {**kw, "residual": kw["residual"][keep]},
               ops.QuantizedRows(want.codes.cpu()[keep], want.scale.cpu()[keep], want.sum.cpu()[keep], want.values.cpu()[keep]))

    def same(got):
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scale.isnan(), want.scale.isnan())
        for a, b in ((got.scale, want.scale), (got.sum, want.sum), (got.values, want.values)):
            assert torch.equal(a[keep.to(DEV)], b[keep.to(DEV)])
        assert bool(got.values[2].isnan().all())
    # outputs of their own
    (bs, total), (bv, values) = (around(torch.zeros(m, k, dtype=dtype), gap, first) for _ in range(2))
    same(ops.quantize_rows(dev(x), **given, sum=total, values=values))
    assert untouched(bs, total) and untouched(bv, values)
    # in place: the values over x, the sum over the residual
    (bx, xs), (br, res) = around(dev(x), gap, first), around(dev(kw["residual"]), gap, first)
    same(ops.quantize_rows(xs, weight=given["weight"], residual=res, sum=res, values=xs))
    assert untouched(bx, xs) and untouched(br, res)
