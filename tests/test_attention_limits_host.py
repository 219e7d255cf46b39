"""Attention's limits, as far as they are refused before the GPU is touched."""
import ctypes

import pytest

from gact.cpp_extension import _abi
from test_attention_adamw_host import EINVAL, Rows, call


@pytest.mark.parametrize("scale,rc", [(3e38, EINVAL), (2.4e38, EINVAL), (2.3e38, 0), (1e-45, 0)])
def test_scales_that_the_exponents_base_takes_to_infinity_are_refused(scale, rc):
    """Scores are multiplied by scale log2(e), as a float: infinite, it makes a NaN of a score of zero."""
    L = _abi.lib()
    a, out = call(batch=0, scale=scale), Rows(16, 4 * 8 * 64, 64, 4 * 64)
    assert L.gact_attention_forward(ctypes.byref(a), ctypes.byref(out), None, None, None, None) == rc
