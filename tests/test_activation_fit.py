"""The polynomial that the layers' kernels of 16-bit types take for the normal distribution's tail, as it stands in their source, against the
error function of the C library: how far it is off is what its comment says."""
import math
import os
import re

import numpy as np

from conftest import ROOT


def tail(a):
    """2 (1 - Phi(a)) in the kernel's float steps (its exponential, within a unit of the last place, exact here)."""
    source = open(os.path.join(ROOT, "gact-icml_amd", "csrc", "layers.hip")).read()
    body = re.search(r"float twice_upper_tail\(float a\) \{(.*?)\n\}", source, re.S).group(1)
    coefficients = [np.float32(c) for c in re.findall(r"(-?\d+\.\d+(?:e-?\d+)?)f", body)]
    assert len(coefficients) == 7
    p = np.full_like(a, coefficients[0])
    for c in coefficients[1:]:
        p = (a.astype(np.float64) * p + np.float64(c)).astype(np.float32)
    return np.exp2((a * p).astype(np.float64))


def test_the_tail_is_as_near_as_it_is_said_to_be():
    a = np.linspace(0, 9, 450001).astype(np.float32)
    got, want = tail(a), np.array([math.erfc(float(v) / math.sqrt(2)) for v in a])
    off = np.abs(got - want)
    for most, bound in ((4, 7.1e-6), (5, 1.1e-5), (6, 2.9e-5), (7, 1.5e-4), (9, 0.03)):
        assert (off <= bound * want)[a <= most].all(), (most, (off / want)[a <= most].max())
    assert want[-1] < 3e-19 and 0.5 * off.max() <= 2.8e-6 and (0.5 * a * off).max() <= 8.3e-7
    # beyond the fit it goes on falling, to nothing
    far = np.concatenate([np.linspace(9, 60, 5001), np.logspace(2, 38, 200)]).astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        beyond = tail(far)
    assert (beyond <= got[-1]).all() and (np.diff(beyond) <= 0).all() and beyond[-1] == 0
