"""CPU checks of the int8 products' sizes at the end of their range: refused before any launch."""

import ctypes

import pytest

from smolvla_mujoco_libero_b200 import _lib as L
from tests.test_answer import _linear


@pytest.mark.parametrize("impl", [L.LINEAR_AUTO, L.LINEAR_FEW, L.LINEAR_MANY])
@pytest.mark.parametrize("m", [1 << 30, 2 ** 31 - 256, 2 ** 31 - 255, 2 ** 31 - 1])
def test_rows_past_30_bits_are_refused(m, impl):
    lib = L.lib()
    assert lib.svla_linear_i8(ctypes.byref(_linear(m=m, impl=impl)), None) == 1
    assert "2^30" in lib.svla_last_error().decode()
