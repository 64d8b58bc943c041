"""The C entries of the attention for training at the ends of sm_scale's range: a backward pass needs at least 2^-100."""
import pytest

from cdna4_sage import _capi
from test_train_cpu import BWD, FWD, P, _err

pytestmark = pytest.mark.skipif(not _capi.LIB_PATH.exists(), reason="libsage_capi.so not built")
STATE = dict(state=P, state_bytes=1 << 20)


@pytest.mark.parametrize("sm", [2.0 ** -101, 2.0 ** -126, 2.0 ** -140])
def test_too_small_for_gradients(sm):
    lib = _capi.lib()
    assert lib.sage_train_fwd(*{**FWD, **STATE, "keep": 1, "sm": sm}.values()) == 2 and "sm_scale" in _err()
    assert lib.sage_train_bwd(*{**BWD, "sm": sm}.values()) == 2 and "sm_scale" in _err()
    # the forward pass alone goes on to its next check
    assert lib.sage_train_fwd(*{**FWD, "sm": sm, "lse": None}.values()) == 1 and "lse" in _err()


@pytest.mark.parametrize("sm,message", [(2.0 ** -100, "lse"), (2.0 ** 127, "lse"), (2.0 ** 127.5, "sm_scale"), (3.4e38, "sm_scale")])
def test_the_ends(sm, message):
    lib = _capi.lib()
    assert lib.sage_train_fwd(*{**FWD, **STATE, "keep": 1, "sm": sm, "lse": None}.values()) == 1 and message in _err()
    assert lib.sage_train_bwd(*{**BWD, "sm": sm, "lse": None}.values()) == 1 and message in _err()
