"""Calls of the decoding operators that are refused for numbers which float32 does not hold, without a GPU."""
import pytest
import torch

import cdna4_sage
from cdna4_sage import _capi
from test_decoding_cpu import ATTN, _err

built = pytest.mark.skipif(not _capi.LIB_PATH.exists(), reason="libsage_capi.so not built")


@pytest.mark.parametrize("sm_scale", [1e-60, 2.0**-149, 2.0**-127, 1e39, float("inf")])
def test_scales_that_float32_does_not_hold_are_refused(sm_scale):
    c = cdna4_sage.new_cache(2, 16, 2, 64, device="cpu")
    with pytest.raises(cdna4_sage.Unsupported, match="sm_scale"):
        cdna4_sage.cache_attention(torch.zeros(1, 4, 2, 64, dtype=torch.float16), c, torch.zeros(1, 2, dtype=torch.int32),
                                   torch.zeros(1, dtype=torch.int32), "NHD", sm_scale)


@built
@pytest.mark.parametrize("sm", [2.0**-149, 2.0**-127, -0.5, float("inf")])
def test_the_entry_refuses_them(sm):
    assert _capi.lib().sage_cache_attn(*{**ATTN, "sm": sm}.values()) == 1 and "sm_scale" in _err()
