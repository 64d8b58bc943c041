"""What the training operators refuse and their host arithmetic, without a GPU."""
import ctypes
from fractions import Fraction

import pytest
import torch

import cdna4_sage
from cdna4_sage import _capi
from train_util import bucket_of

built = pytest.mark.skipif(not _capi.LIB_PATH.exists(), reason="libsage_capi.so not built")
P = 0x10000  # an aligned address that is never read: the checks come first


def _err():
    return _capi.lib().sage_last_error().decode()


# ---- borders of the buckets -----------------------------------------------------------------------------------------------

@built
@pytest.mark.parametrize("buckets,two,reach", [(32, True, 128), (32, False, 128), (4, True, 2), (2, False, 3), (64, True, 800),
                                               (255, False, 129), (256, True, 5000), (256, False, 2 ** 30 - 1), (16, True, 9),
                                               (128, False, 65)])
def test_borders_are_exact(buckets, two, reach):
    side = buckets // 2 if two else buckets
    near, m = side // 2, side - side // 2
    got = list(_capi.bias_borders(buckets, two, reach))
    assert got[0] == near and len(got) == m
    for t, n in enumerate(got):
        # the smallest n with (n / near)^m >= (reach / near)^t
        def reached(n):
            return Fraction(n, near) ** m >= Fraction(reach, near) ** t
        assert reached(n) and (n == 1 or not reached(n - 1))
    assert got[-1] <= reach
    for n in list(range(0, min(got[-1] + 3, 400))) + got + [reach, 2 * reach]:
        b = max([x for x in range(m) if got[x] <= n], default=-1)
        assert bucket_of(-n, buckets, reach, two) == (n if n < near else near + b)


@built
@pytest.mark.parametrize("buckets,two,reach", [(32, True, 8), (1, False, 9), (257, False, 900), (6, True, 1), (5, True, 9), (2, True, 9),
                                               (32, False, 2 ** 30)])
def test_borders_refuse(buckets, two, reach):
    out = (ctypes.c_int * 256)()
    assert _capi.lib().sage_bias_borders(buckets, int(two), reach, out) == _capi.SAGE_ERR_INVALID and _err()


# ---- the Python layer -----------------------------------------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16)
    U = cdna4_sage.Unsupported
    with pytest.raises(U, match="GPU"):
        cdna4_sage.attention_train(q, q, q)
    with pytest.raises(U, match="GPU"):
        cdna4_sage.attention_train_varlen(q[0], q[0], q[0], torch.tensor([0, 2]), torch.tensor([0, 2]))
    with pytest.raises(U, match="GPU"):
        cdna4_sage.relative_bias(torch.zeros(32, 2), 3, 3)


def test_refusals_before_the_device_is_looked_at():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    f, U = cdna4_sage.attention_train, cdna4_sage.Unsupported
    q = z(1, 2, 8, 64)
    for call, message in ((lambda: f(q, q, q, "BHSD"), "layout"), (lambda: f(q[0], q, q), "4D"),
                          (lambda: f(z(1, 2, 8, 64, dtype=torch.float32), q, q), "dtype"), (lambda: f(q, q, z(1, 2, 9, 64)), "one shape"),
                          (lambda: f(z(1, 2, 8, 80), z(1, 2, 8, 80), z(1, 2, 8, 80)), "head_dim"),
                          (lambda: f(z(1, 3, 8, 64), q, q), "multiple"), (lambda: f(z(2, 2, 8, 64), q, q), "batch"),
                          (lambda: f(q, q, q, sm_scale=2.0 ** -140), "sm_scale")):
        with pytest.raises(U, match=message):
            call()
    g = cdna4_sage.attention_train_varlen
    cu = torch.tensor([0, 8], dtype=torch.int32)
    for bad in ((cu[:1], cu[:1]), (cu, torch.tensor([0, 4, 8])), (cu[None], cu[None])):
        with pytest.raises(U, match="cu_seqlens"):
            g(q[0], q[0], q[0], *bad)
    with pytest.raises(U, match="3D"):
        g(q, q, q, cu, cu)


# ---- the C entries --------------------------------------------------------------------------------------------------------

def _ints(*x):
    return (ctypes.c_int * len(x))(*x)


T = lambda n: {f"{n}": P, f"{n}b": 8 * 64 * 2, f"{n}s": 64 * 2, f"{n}h": 64}  # noqa: E731
SIZES = dict(B=1, H=2, Hkv=2, Sq=8, Skv=8, D=64, dtype=0, causal=0, sm=0.0, cu_q=None, cu_k=None)
FWD = dict(**T("q"), **T("k"), **T("v"), **T("o"), lse=P, **SIZES, mask=None, msb=0, msh=0, msq=0, msk=0, table=None, tdtype=0, tb=0,
           th=0, buckets=0, two=0, borders=None, keep=0, state=None, state_bytes=0, stream=None)
BWD = dict(**T("g"), **T("q"), **T("k"), **T("v"), **T("o"), lse=P, **T("dq"), **T("dk"), **T("dv"), **SIZES, has_mask=0, msb=0, msh=0,
           msq=0, dtable=None, tdtype=0, tb=0, th=0, buckets=0, two=0, borders=None, state=P, state_bytes=1 << 20, ws=P, ws_bytes=1 << 20, stream=None)
COMMON = [
    (dict(q=None), 1, "q is NULL"), (dict(k=P + 8), 1, "k must be"), (dict(vs=7), 1, "v must be"), (dict(lse=None), 1, "lse"),
    (dict(H=3), 1, "multiple"), (dict(D=80), 2, "head_dim 80"), (dict(dtype=2), 2, "dtype"), (dict(Sq=0), 1, "positive"),
    (dict(sm=-1.0), 1, "sm_scale"), (dict(sm=float("nan")), 1, "sm_scale"), (dict(sm=float("inf")), 1, "sm_scale"),
    (dict(cu_q=P), 1, "go together"), (dict(cu_q=P, cu_k=P, state=None), 1, "state"),
    (dict(buckets=32, borders=None), 1, "borders"), (dict(buckets=1, borders=_ints(1)), 1, "buckets"),
    (dict(buckets=4, two=1, borders=_ints(5)), 1, "borders"),
    (dict(buckets=4, borders=_ints(2, 1)), 1, "must not fall"),
    (dict(buckets=4, borders=_ints(2, 900)), 2, "distance 900"), (dict(buckets=4, borders=_ints(2, 5), tdtype=2), 1, "table dtype"),
]


@built
@pytest.mark.parametrize("change,code,message", COMMON + [
    (dict(o=None), 1, "out is NULL"), (dict(mask=P), 1, "state"), (dict(keep=1), 1, "state"), (dict(mask=P, cu_q=P, cu_k=P), 1, "no mask"),
    (dict(buckets=4, borders=_ints(2, 5), state=P, state_bytes=1 << 20), 1, "table is NULL"),
    (dict(mask=P, state=P + 16, state_bytes=1 << 20), 1, "256-byte"),
])
def test_forward_entry_refuses(change, code, message):
    assert _capi.lib().sage_train_fwd(*{**FWD, **change}.values()) == code and message in _err(), _err()


@built
@pytest.mark.parametrize("change,code,message", COMMON + [
    (dict(g=None), 1, "dout is NULL"), (dict(dqs=4), 1, "dq must be"), (dict(dk=None), 1, "go together"), (dict(ws=None), 1, "workspace"),
    (dict(ws_bytes=100), 1, "workspace"), (dict(dq=None, dk=None, dv=None), 1, "no gradient"), (dict(dq=None, dtable=P), 1, "dtable"),
    (dict(state=None), 1, "state"), (dict(state=P + 16), 1, "256-byte"),
])
def test_backward_entry_refuses(change, code, message):
    assert _capi.lib().sage_train_bwd(*{**BWD, **change}.values()) == code and message in _err(), _err()


@built
def test_bias_entries_refuse():
    b = _capi.bias_borders(32, True, 128)
    ok = dict(table=P, tdtype=3, tb=2, th=1, H=2, buckets=32, two=1, borders=b, q=4, k=4, offset=0, at=None, o64=0, out=P, dtype=0, stream=None)
    for change, message in ((dict(table=None), "NULL"), (dict(tdtype=2), "table dtype"), (dict(dtype=2), "dtype"), (dict(H=0), "heads"),
                            (dict(q=0), "positive"), (dict(out=P + 1), "misaligned"), (dict(at=P + 4, o64=1), "misaligned"),
                            (dict(borders=None), "borders"), (dict(buckets=31), "buckets")):
        assert _capi.lib().sage_relative_bias(*{**ok, **change}.values()) == 1 and message in _err(), _err()
    ok = dict(d=P, sh=16, sq=4, dtype=0, H=2, buckets=32, two=1, borders=b, q=4, k=4, offset=0, at=None, o64=0, dt=P, tdtype=3, tb=2, th=1,
              ws=P, ws_bytes=1 << 20, stream=None)
    for change, message in ((dict(d=None), "NULL"), (dict(dt=None), "NULL"), (dict(ws=None), "NULL"), (dict(ws_bytes=8), "workspace"),
                            (dict(d=P + 1), "misaligned"), (dict(k=-1), "positive"), (dict(dtype=2), "dtype")):
        assert _capi.lib().sage_relative_bias_grad(*{**ok, **change}.values()) == 1 and message in _err(), _err()


@built
def test_workspaces():
    """Sizes follow from the shapes alone: none without masks, bias or packing; a mask costs its bits and little more."""
    ws = _capi.train_workspace
    state, work = ws(False, 2, 8, 8, 1000, 1000, 64, None, None, False)
    assert state == 0 and ws(False, 2, 8, 8, 1000, 1000, 64, None, None, True)[0] == 2 * 8 * 1000 * 64 * 2 and work >= 2 * 4 * 2 * 8 * 1024
    assert ws(False, 2, 8, 8, 1000, 1000, 64, (0, 0, 0), None, False)[0] <= 2048
    full = ws(False, 2, 8, 8, 1000, 1000, 64, (1, 1, 1), None, False)[0]
    assert 2 * 8 * 1024 * 1024 // 8 <= full <= 1.1 * 2 * 8 * 1024 * 1024 // 8
    assert ws(True, 5, 8, 8, 1000, 900, 64, None, None, False)[0] > 0
    assert ws(False, 2, 8, 8, 1000, 1000, 64, None, (32, True, 128), False)[0] >= 8 * 183 * 4
    with pytest.raises(_capi.SageError, match="distance"):
        ws(False, 2, 8, 8, 1000, 1000, 64, None, (32, True, 2000), False)
