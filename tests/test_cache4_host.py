"""Limits of the 4-bit cache's operators that the host checks, one step to either side where nothing need launch."""
import math

import numpy as np
import pytest

from fbsa_amd import _lib
from test_cache4_refusals import _attn


@pytest.mark.parametrize("sign", [1, -1])
def test_scales_up_to_2_127(sign):
    """Rows of very large scores take the power of two at or above the scale times log2(e), which has to be a number."""
    lib, log2e = _lib.load(), np.float32(1.4426950408889634)
    most = np.float32(2.0 ** 127 / 1.4426950408889634)
    while most * log2e > np.float32(2.0 ** 127):
        most = np.nextafter(most, np.float32(0))
    over = most
    while over * log2e <= np.float32(2.0 ** 127):
        over = np.nextafter(over, np.float32(math.inf))
    assert lib.fbsa_cache4_attn_workspace_bytes(_attn(scale=sign * float(most))) > 0
    assert lib.fbsa_cache4_attn_workspace_bytes(_attn(scale=sign * float(over))) == 0
    assert "scale" in lib.fbsa_last_error().decode()
