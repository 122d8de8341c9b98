"""CPU checks of the serving operators at the edge of what they take: arguments that would give a wrong answer or leave the
kernels' index arithmetic are refused before any launch."""

import ctypes
import math

import pytest

from smolvla_mujoco_libero_b200 import _lib as L
from smolvla_mujoco_libero_b200 import ops
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
