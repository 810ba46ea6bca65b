"""Scales that leave the fp32 range once they count in powers of two are refused by the 8-bit cache's attention."""
import ctypes

import pytest

from flashact_amd import _lib
from tests.test_kv8 import _attn_args


@pytest.mark.parametrize("kw", [dict(scale=3e38), dict(scale=-3e38), dict(softcap=3e38)])
def test_scales_past_the_range_are_refused(kw):
    lib = _lib.lib()
    assert lib.fa_kv8_attention(ctypes.byref(_attn_args(**kw)), None) == 1
    assert "fp32 range" in lib.fa_last_error().decode()
