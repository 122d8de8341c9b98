"""CPU checks of the serving operators at the edge of what they take: arguments that would give a wrong answer or leave the
kernels' index arithmetic are refused before any launch."""

import ctypes
import math

import pytest
import torch

from oracle import serving as S
from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import build, ops
from tests.test_serving import _packed, _paged


@pytest.mark.parametrize("scale", [-0.125, -1e-30, math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("name,make", [("svla_packed_attention", _packed), ("svla_paged_attention", _paged)])
def test_scales_that_do_not_fit_are_refused(name, make, scale):
    lib = L.lib()
    assert getattr(lib, name)(ctypes.byref(make(scale=scale)), None) == 1
    assert "scale" in lib.svla_last_error().decode()


@pytest.mark.parametrize("table", [ops.rope_table, ops.rope_table_wide])
def test_rotation_tables_are_made_on_a_gpu_only(table):
    with pytest.raises(ValueError, match="CUDA"):
        table(16, 10000.0, "cpu")


def test_tables_that_reach_past_31_bits_are_refused():
    """Entries are numbered in 32 bits, and a tile's last one may lie up to 63 behind the sequence's."""
    lib = L.lib()
    for pages, page in ((1 << 23, 256), (1 << 27, 16), ((1 << 31) - 1, 256)):
        d = _paged(max_pages=pages, page_size=page, page_table_rs=1 << 31)
        assert lib.svla_paged_attention(ctypes.byref(d), None) == 1
        assert "max_pages" in lib.svla_last_error().decode()


@pytest.mark.parametrize("offset,spread", [(100.0, 1.0), (-100.0, 1.0), (1000.0, 0.5), (0.0, 1.0)])
def test_plain_quantisation_of_groups_with_an_offset(offset, spread):
    """step / 2 + |low| 2^-8 + 15 step 2^-8, as the header states it.  Both pairs enter rounded: by at most 2^-8 of
    themselves, which 1 / (1 - 2^-8) covers; 1e-6 of the size for fp32's own roundings."""
    x = offset + spread * torch.rand(200, 128, generator=torch.Generator().manual_seed(6))
    codes, step, low = S.quantise(x)
    err = (S.held(codes, step, low) - x).abs().unflatten(-1, (-1, 32))
    s, m = step.float().unsqueeze(-1), low.float().abs().unsqueeze(-1)
    bound = s / 2 + (m + 15 * s) * 2.0 ** -8 / (1 - 2.0 ** -8) + 1e-6 * (m + 15 * s)
    assert bool((err <= bound).all())
    if offset:  # the offset costs whole steps
        assert float((err / s).max()) > 2


def test_plain_quantisation_of_a_range_beyond_fp32():
    x = torch.zeros(1, 64)
    x[0, 0], x[0, 1] = -3e38, 3e38
    held = S.held(*S.quantise(x))
    assert bool(torch.isnan(held[0, :32]).all()) and bool((held[0, 32:] == 0).all())


def test_module_of_another_torch_is_noticed(monkeypatch):
    """The torch side is bound to the torch and the Python it was built with: another one's is rebuilt by the build, and
    refused, not loaded, at the first call."""
    assert build.torch_module_fits()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    assert not build.torch_module_fits() and not build.up_to_date()
    monkeypatch.setattr(L, "_serving", None)
    with pytest.raises(L.SvlaError, match="another torch"):
        L.serving()
