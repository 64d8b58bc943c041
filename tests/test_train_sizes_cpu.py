"""How many sequences and heads the attention for training takes: what a launch of its kernels holds, and no less."""
import pytest
import torch

import cdna4_sage
from cdna4_sage import _capi, _train

pytestmark = pytest.mark.skipif(not _capi.LIB_PATH.exists(), reason="libsage_capi.so not built")


def _sizes(packed, B, H, Hkv, Sq, Skv, D, mask=None):
    cu = torch.empty(B + 1, device="meta") if packed else None
    return _train._sizes((B, H, Hkv, Sq, Skv, D, 0), None, mask, cu, True)


@pytest.mark.parametrize("packed,B,H,Hkv,Sq,Skv,D", [
    (False, 8192, 16, 16, 64, 64, 64), (False, 65536, 64, 8, 100, 128, 128), (False, 1, 128, 128, 1 << 20, 1 << 20, 128),
    (False, 32767, 255, 255, 7, 9, 256), (False, 262080, 64, 64, 1, 1, 96),
    (True, 4096, 32, 8, 524288, 524288, 128), (True, 100000, 64, 64, 1 << 20, 1 << 20, 64), (True, 8192, 128, 16, 8192, 1 << 20, 256),
])
def test_sizes_that_fit_are_taken(packed, B, H, Hkv, Sq, Skv, D):
    state, work, batch = _sizes(packed, B, H, Hkv, Sq, Skv, D)
    rows = (1 if packed else B) * H * Sq
    assert state >= 2 * rows * D and work >= 8 * rows and batch == B


@pytest.mark.parametrize("packed,B,H,Hkv,Sq,Skv,D", [
    (False, 65536, 256, 256, 64, 64, 64), (False, 65536, 128, 128, 64, 64, 256), (False, 65536, 128, 128, 129, 1, 128),
    (False, 65536, 128, 128, 1, 129, 128), (False, 262144, 64, 64, 1, 1, 64), (True, 300000, 64, 64, 1, 1, 128),
    (True, 1, 64, 64, 1 << 25, 1, 64), (False, 1 << 24, 1, 1, 1, 1, 64), (False, 1, 1 << 16, 1, 1, 1, 64),
])
def test_sizes_that_do_not_are_refused(packed, B, H, Hkv, Sq, Skv, D):
    with pytest.raises(cdna4_sage.Unsupported, match="too"):
        _sizes(packed, B, H, Hkv, Sq, Skv, D)


def test_masks():
    assert _sizes(False, 2, 8, 8, 100000, 100000, 64, (0, 0, 1))[0] >= 100000 * 100000 // 8
    assert _sizes(False, 512, 64, 64, 4096, 4096, 64, (0, 0, 1))
    with pytest.raises(cdna4_sage.Unsupported, match="mask too large"):
        _sizes(False, 128, 64, 64, 4096, 4096, 64, (1, 1, 1))
