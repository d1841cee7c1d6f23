"""Scales whose product with log2 e, which the attention kernels take, leaves fp32 are refused:
every weight would be a NaN. (Host pointers: nothing is launched.)"""

import os

import numpy as np
import pytest

from param_decomp_amd import _lib as L

pytestmark = pytest.mark.skipif(not os.path.exists(L.LIB_PATH), reason="HIP library not built")


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scales_at_the_end_of_fp32_are_refused(scale):
    raw = np.zeros(4096, np.uint8)
    p = (raw.ctypes.data + 63) // 64 * 64
    head = [p, 64, 16, p, 32, 16, p, 32, 16, 1, 4, 4, 2, 16, p, 1, scale, 1]
    with pytest.raises(L.PDError, match="scale"):
        L.call("pd_packed_attention_fwd", *head, p, None, p, None)
    with pytest.raises(L.PDError, match="scale"):
        L.call("pd_packed_attention_bwd", *head, p, p, p, p, p, p, p, p, 1 << 30, None)
