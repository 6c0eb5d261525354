"""CPU tests: the scales that attention takes.  The kernels multiply by scale * log2(e) in FP32."""

from __future__ import annotations

import numpy as np
import pytest

from testfiles_b200 import _native
from test_paged_refusals import attend

LARGEST = float(np.float32(3.4028234663852886e38) / np.float32(1.4426950408889634))


@pytest.mark.parametrize("scale", [0.0, -0.0, 2.9e38, 3.0e38, LARGEST * 1.000001, 3.4028234663852886e38])
def test_scales_that_are_none_or_overflow(scale):
    assert attend(scale=scale, hk=1) == _native.ERR_BAD_MODE


@pytest.mark.parametrize("scale", [1.5e-45, 1e-30, 1 / 16, 1e30, LARGEST * 0.999999])
def test_scales_that_are_taken(scale):
    assert np.float32(scale) > 0 and np.isfinite(np.float32(scale) * np.float32(1.4426950408889634))
    assert attend(scale=scale, n=0, b=0) == _native.OK
