"""What the decoding operators refuse and their host arithmetic, without a GPU."""
import ctypes
import math

import pytest
import torch

import cdna4_sage
from cdna4_sage import _cache, _capi, _rope

built = pytest.mark.skipif(not _capi.LIB_PATH.exists(), reason="libsage_capi.so not built")
P = 0x10000  # an aligned address that is never read: the checks come first


def _err():
    return _capi.lib().sage_last_error().decode()


# ---- frequencies and slots --------------------------------------------------------------------------------------------

def test_frequencies():
    f, c = cdna4_sage.rope_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,) and c == 1.0
    assert f[0] == 1.0 and abs(float(f[16]) - 0.01) < 1e-15
    lin, _ = cdna4_sage.rope_frequencies(64, scaling={"type": "linear", "factor": 4})
    assert torch.allclose(lin * 4, f, rtol=1e-15)
    ntk, _ = cdna4_sage.rope_frequencies(64, scaling={"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and abs(float(ntk[-1] / f[-1]) - 0.25) < 1e-12
    y, c = cdna4_sage.rope_frequencies(64, scaling={"type": "yarn", "factor": 4, "original_length": 2048})
    turns = 2048 * f / (2 * math.pi)
    assert abs(c - (0.1 * math.log(4) + 1)) < 1e-15
    assert torch.equal(y[turns > 32 * 2], f[turns > 32 * 2])
    assert torch.allclose(y[turns < 0.5], f[turns < 0.5] / 4, rtol=1e-15)
    assert bool((y <= f).all()) and bool((y >= f / 4 * (1 - 1e-15)).all())
    assert cdna4_sage.rope_frequencies(64, scaling={"type": "yarn", "factor": 4, "original_length": 99,
                                                    "attention_factor": 1.0})[1] == 1.0
    for bad in ({"type": "linear"}, {"type": "other", "factor": 2}, {"type": "linear", "factor": 0.5},
                {"type": "yarn", "factor": 2}, {"type": "linear", "factor": float("nan")}):
        with pytest.raises(ValueError):
            cdna4_sage.rope_frequencies(64, scaling=bad)
    for rot in (0, 7, -2):
        with pytest.raises(ValueError):
            cdna4_sage.rope_frequencies(rot)


def test_slots():
    table = torch.tensor([[3, 0, -1], [2, 5, 7]], dtype=torch.int32)
    got = cdna4_sage.cache_slots(table, torch.tensor([34, 2]), 4, 16)
    assert got.tolist() == [[14, 15, -1, -1], [-1, -1, 32, 33]]
    got = cdna4_sage.cache_slots(table, torch.tensor([50, 48], dtype=torch.int32), 3, 16)
    assert got.tolist() == [[-1, -1, -1], [7 * 16 + 13, 7 * 16 + 14, 7 * 16 + 15]]
    assert cdna4_sage.cache_slots(table[:, :0], torch.tensor([1, 2]), 2, 16).tolist() == [[-1, -1], [-1, -1]]
    assert cdna4_sage.cache_slots(table, torch.tensor([1, 2]), 0, 16).shape == (2, 0)
    with pytest.raises(cdna4_sage.Unsupported):
        cdna4_sage.cache_slots(table, torch.tensor([1, 2]), 1, 24)


# ---- the Python layer's refusals --------------------------------------------------------------------------------------

def _cpu_cache(pages=2, n=16, heads=2, D=64, dtype=torch.int8):
    return cdna4_sage.new_cache(pages, n, heads, D, dtype, device="cpu")


def test_new_cache():
    c = _cpu_cache(3, 32, 4, 96, torch.float8_e4m3fn)
    assert c.k.shape == (3, 4, 32, 96) and c.k.dtype == torch.float8_e4m3fn and c.v_scale.shape == (3, 4, 32)
    assert not bool(c.k.view(torch.int8).any()) and not bool(c.k_scale.any())
    for bad in (dict(n=24), dict(n=8), dict(n=2048), dict(D=80), dict(dtype=torch.uint8), dict(pages=0), dict(heads=0)):
        with pytest.raises(cdna4_sage.Unsupported):
            _cpu_cache(**bad)


@pytest.mark.parametrize("call", [
    lambda c, q: cdna4_sage.cache_write(c, q[0], q[0], torch.zeros(4, dtype=torch.int64)),
    lambda c, q: cdna4_sage.cache_read(c, torch.zeros(4, dtype=torch.int64)),
    lambda c, q: cdna4_sage.cache_attention(q, c, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), "NHD"),
    lambda c, q: cdna4_sage.rope(q, None, None, cdna4_sage.rope_frequencies(64)[0], "NHD"),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(cdna4_sage.Unsupported):
        call(_cpu_cache(), torch.zeros(1, 4, 2, 64, dtype=torch.float16))


def test_refusals_before_the_device_is_looked_at():
    c, z = _cpu_cache(), torch.zeros(4, dtype=torch.int64)
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    for k, v, s, layout in ((x, x[:3], z, "HND"), (x.float(), x.float(), z, "HND"), (x, x.bfloat16(), z, "HND"),
                            (x, x, z, "BHSD"), (x[0], x[0], z, "HND")):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.cache_write(c, k, v, s, layout)
    for dtype, layout in ((torch.float32, "HND"), (torch.int8, "HND"), (torch.float16, "other")):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.cache_read(c, z, dtype, layout)
    q, f = torch.zeros(1, 4, 2, 64, dtype=torch.float16), cdna4_sage.rope_frequencies(64)[0]
    bad = [dict(q=q.float()), dict(q=q[0]), dict(freqs=None), dict(freqs=f.float()), dict(freqs=f[:0]), dict(freqs=f[:3]),
           dict(freqs=cdna4_sage.rope_frequencies(72)[0]), dict(positions=torch.zeros(4)), dict(positions=z[:3]),
           dict(positions=z.view(2, 2)), dict(k=q[:, :3]), dict(k=q.bfloat16()), dict(k=q[..., :32]),
           dict(tensor_layout="x"), dict(q=torch.zeros(1, 4, 2, 80, dtype=torch.float16))]
    for kw in bad:
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.rope(**{**dict(q=q, k=None, positions=None, freqs=f, tensor_layout="NHD"), **kw})


def test_cache_tensors_that_do_not_fit_are_refused():
    c = _cpu_cache()
    wrong = [c._replace(v=c.v[:1]), c._replace(k_scale=c.k_scale[..., :8]), c._replace(k_scale=c.k_scale.half()),
             c._replace(v=c.v.view(torch.float8_e4m3fn)), c._replace(k=c.k.to(torch.uint8), v=c.v.to(torch.uint8)),
             c._replace(k=c.k[0]), c._replace(k=c.k.transpose(1, 2).contiguous().transpose(1, 2)),
             cdna4_sage.KVCache(*(t[:, :, :8].contiguous() for t in c)), cdna4_sage.KVCache(*(t[:0] for t in c)), c]
    for x in wrong:   # (the last one is refused for being on the CPU)
        with pytest.raises(cdna4_sage.Unsupported):
            _cache.check_cache(x)


# ---- the C entries' refusals ------------------------------------------------------------------------------------------

ROPE = dict(q=P, qsb=4096, qss=256, qsh=64, qo=P, qob=4096, qos=256, qoh=64, H=4, k=P, ksb=4096, kss=128, ksh=64, ko=P,
            kob=4096, kos=128, koh=64, Hk=2, B=1, S=4, D=64, dtype=0, pos=P, p64=1, psb=0, pss=1, freqs=P, rot=64,
            inter=0, factor=1.0, inverse=0, stream=None)


@built
@pytest.mark.parametrize("change,code,message", [
    (dict(q=None), 1, "NULL"), (dict(qo=None), 1, "NULL"), (dict(freqs=None), 1, "NULL"), (dict(k=None), 1, "NULL"),
    (dict(ko=None), 1, "NULL"), (dict(B=0), 1, "positive"), (dict(S=-1), 1, "positive"), (dict(H=0), 1, "positive"),
    (dict(Hk=-1), 1, "positive"), (dict(dtype=2), 2, "dtype"), (dict(D=80), 2, "head_dim"), (dict(rot=0), 2, "rotated"),
    (dict(rot=12), 2, "rotated"), (dict(rot=72), 2, "rotated"), (dict(q=P + 2), 1, "aligned"), (dict(ko=P + 8), 1, "aligned"),
    (dict(qss=250), 1, "strides"), (dict(koh=4), 1, "strides"), (dict(pos=P + 4), 1, "misaligned"),
    (dict(freqs=P + 4), 1, "misaligned"), (dict(B=1 << 20, S=1 << 20), 1, "too many")])
def test_rope_entry_refuses(change, code, message):
    assert _capi.lib().sage_rope(*{**ROPE, **change}.values()) == code
    assert message in _err()


WRITE = dict(k=P, ksb=0, kss=128, ksh=64, v=P, vsb=0, vss=128, vsh=64, B=1, S=4, dtype=0, slots=P, s64=1, k8=P, ks=P, v8=P,
             vs=P, pages=2, n=16, Hkv=2, D=64, ct=0, stream=None)


@built
@pytest.mark.parametrize("change,code,message", [
    (dict(k=None), 1, "NULL"), (dict(slots=None), 1, "NULL"), (dict(k8=None), 1, "NULL"), (dict(vs=None), 1, "NULL"),
    (dict(v=P + 8), 1, "aligned"), (dict(v8=P + 8), 1, "aligned"), (dict(ks=P + 4), 1, "aligned"),
    (dict(slots=P + 4), 1, "misaligned"), (dict(kss=100), 1, "strides"), (dict(B=0), 1, "positive"),
    (dict(pages=0), 1, "positive"), (dict(Hkv=0), 1, "positive"), (dict(n=24), 2, "page_size"), (dict(n=8), 2, "page_size"),
    (dict(n=2048), 2, "page_size"), (dict(D=80), 2, "head_dim"), (dict(ct=2), 2, "cache dtype"), (dict(dtype=2), 2, "dtype"),
    (dict(B=1 << 20, S=1 << 20), 1, "too many"), (dict(B=1 << 14, S=1 << 14, Hkv=9), 1, "too many")])
@pytest.mark.parametrize("entry", ["sage_cache_write", "sage_cache_read"])
def test_cache_entries_refuse(entry, change, code, message):
    assert getattr(_capi.lib(), entry)(*{**WRITE, **change}.values()) == code
    assert message in _err() and entry in _err()


ATTN = dict(q=P, qsb=512, qss=512, qsh=64, out=P, osb=512, oss=512, osh=64, lse=None, k8=P, ks=P, v8=P, vs=P, table=P,
            ts=4, lengths=P, tree=None, msb=0, msq=0, msk=0, B=1, H=8, Hkv=2, T=1, D=64, dtype=0, ct=0, pages=4, n=16,
            max_pages=4, causal=1, sm=0.0, ws=P, wsb=1 << 40, stream=None)


@built
@pytest.mark.parametrize("change,code,message", [
    (dict(q=None), 1, "NULL"), (dict(table=None), 1, "NULL"), (dict(lengths=None), 1, "NULL"), (dict(v8=None), 1, "NULL"),
    (dict(q=P + 2), 1, "aligned"), (dict(out=P + 8), 1, "aligned"), (dict(lengths=P + 2), 1, "misaligned"),
    (dict(qsh=60), 1, "strides"), (dict(B=0), 1, "positive"), (dict(T=0), 1, "positive"), (dict(max_pages=0), 1, "positive"),
    (dict(H=7), 1, "multiple"), (dict(D=80), 2, "head_dim"), (dict(n=20), 2, "page_size"), (dict(dtype=2), 2, "dtype"),
    (dict(ct=7), 2, "cache dtype"), (dict(sm=-1.0), 1, "sm_scale"), (dict(sm=float("nan")), 1, "sm_scale"),
    (dict(sm=float("inf")), 1, "sm_scale"), (dict(n=1024, max_pages=1 << 21), 1, "2^30"), (dict(T=1 << 28), 1, "2^28"),
    (dict(B=1 << 18, n=1024, max_pages=1 << 20), 1, "2^37"), (dict(T=9, tree=P, msq=1 << 28), 1, "tree mask"),
    (dict(T=9, tree=P, msk=-(1 << 40)), 1, "tree mask")])
def test_attention_entry_refuses(change, code, message):
    assert _capi.lib().sage_cache_attn(*{**ATTN, **change}.values()) == code
    assert message in _err()


@built
def test_attention_workspace_refuses():
    ws = ctypes.c_int64(-1)
    assert _capi.lib().sage_cache_attn_workspace(1, 8, 2, 1, 64, 16, 4, None) == 1
    assert _capi.lib().sage_cache_attn_workspace(1, 7, 2, 1, 64, 16, 4, ctypes.byref(ws)) == 1 and ws.value == -1
