"""cdna4_sage.attention_train and attention_train_varlen against float64: outputs, logsumexp and gradients over head dims, types,
layouts, lengths from one token on, shared heads, masks that leave rows empty, packed sequences and the bias inside."""
import math

import pytest
import torch

import cdna4_sage
from train_util import Exact, bucket_map, close

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _draw(B, H, Hkv, Sq, Skv, D, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, H, Sq, D, generator=g) * scale
    k, v = (torch.randn(B, Hkv, Skv, D, generator=g) for _ in range(2))
    k = k + torch.randn(D, generator=g) * (torch.rand(D, generator=g) < 0.1)
    do = torch.randn(B, H, Sq, D, generator=g)
    return [t.to(dtype) for t in (q, k, v, do)]


def _put(t, layout, dev):
    return (t if layout == "HND" else t.transpose(1, 2).contiguous()).to(dev)


def _hnd(t, layout):
    return t if layout == "HND" else t.transpose(1, 2)


def _run(dev, q, k, v, do, layout="HND", table=None, **kw):
    leaves = [_put(t, layout, dev).requires_grad_() for t in (q, k, v)]
    more = {}
    if table is not None:
        more["bias_table"] = table.detach().to(dev).requires_grad_()
        leaves.append(more["bias_table"])
    out, lse = cdna4_sage.attention_train(*leaves[:3], tensor_layout=layout, return_lse=True, **more, **kw)
    assert out.dtype == q.dtype and out.shape == leaves[0].shape and not lse.requires_grad
    grads = torch.autograd.grad(out, leaves, _put(do, layout, dev))
    for a, b in zip(grads, leaves):
        assert a.dtype == b.dtype and a.shape == b.shape
    return _hnd(out, layout), lse, [_hnd(t, layout) if t.dim() == 4 else t for t in grads]


def _compare(e, out, lse, grads):
    close(out, e.out, e.room_out)
    empty = e.lse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    close(torch.where(empty, 0.0, lse.cpu()), torch.where(empty, 0.0, e.lse), e.room_lse)
    for got, want, room in zip(grads, (e.dq, e.dk, e.dv), (e.room_dq, e.room_dk, e.room_dv)):
        close(got, want, room)


CASES = [
    # B, H, Hkv, Sq, Skv, D, dtype, layout, causal
    (1, 1, 1, 1, 1, 64, BF, "HND", False),
    (2, 2, 1, 1, 700, 128, BF, "NHD", True),
    (1, 2, 2, 33, 1, 96, HF, "HND", False),
    (2, 3, 3, 64, 64, 64, HF, "NHD", True),
    (1, 4, 2, 65, 129, 128, BF, "HND", True),
    (2, 2, 2, 128, 128, 256, BF, "NHD", False),
    (1, 6, 2, 257, 300, 96, BF, "HND", True),
    (1, 2, 1, 300, 130, 128, HF, "NHD", True),      # queries before the first key see nothing
    (1, 2, 1, 300, 130, 256, BF, "HND", True),
    (2, 8, 1, 191, 513, 64, BF, "NHD", True),
    (1, 4, 4, 500, 77, 128, HF, "HND", False),
    (1, 4, 1, 333, 450, 256, HF, "NHD", True),
    (3, 5, 5, 130, 259, 96, HF, "NHD", False),
    (1, 2, 2, 1025, 1100, 128, BF, "HND", True),
]


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D,dtype,layout,causal", CASES)
def test_matches_float64(dev, B, H, Hkv, Sq, Skv, D, dtype, layout, causal):
    q, k, v, do = _draw(B, H, Hkv, Sq, Skv, D, dtype)
    out, lse, grads = _run(dev, q, k, v, do, layout, is_causal=causal)
    _compare(Exact(q, k, v, causal=causal, dout=do), out, lse, grads)
    again = _run(dev, q, k, v, do, layout, is_causal=causal)
    assert torch.equal(out, again[0]) and all(torch.equal(a, b) for a, b in zip(grads, again[2]))
    plain = cdna4_sage.attention_train(*(_put(t, layout, dev) for t in (q, k, v)), tensor_layout=layout, is_causal=causal)
    assert torch.equal(_hnd(plain, layout), out) and plain.grad_fn is None


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("sm_scale,spread", [(0.5, 3.0), (0.02, 1.0), (1.0, 8.0)])
def test_scales_and_sharp_rows(dev, dtype, sm_scale, spread):
    """Large scores: weights from 1 down to nothing."""
    q, k, v, do = _draw(1, 2, 2, 200, 333, 64, dtype, seed=4, scale=spread)
    out, lse, grads = _run(dev, q, k, v, do, sm_scale=sm_scale)
    _compare(Exact(q, k, v, dout=do, sm_scale=sm_scale), out, lse, grads)
    for default in (None, 0.0, -1.0, float("nan")):
        a = cdna4_sage.attention_train(q.to(dev), k.to(dev), v.to(dev), sm_scale=default)
        assert torch.equal(a, cdna4_sage.attention_train(q.to(dev), k.to(dev), v.to(dev)))


@pytest.mark.parametrize("size", [2.0 ** -14, 1.0, 2.0 ** 12])
def test_gradients_of_any_size_in_fp16(dev, size):
    """A loss scaled far up or down: fp16's gradients keep their precision as long as they are themselves in its range."""
    q, k, v, do = _draw(1, 2, 1, 150, 180, 64, HF, seed=6)
    do = (do.float() * size).to(HF)
    v = (v.float() / max(1.0, size / 16)).to(HF)
    out, lse, grads = _run(dev, q, k, v, do)
    e = Exact(q, k, v, dout=do)
    smallest = 2.0 ** -25     # half of fp16's smallest step, where a gradient itself is subnormal
    close(grads[0], e.dq, e.room_dq + smallest)
    close(grads[1], e.dk, e.room_dk + smallest)
    close(grads[2], e.dv, e.room_dv + smallest)


def _docs(S, sizes):
    d = []
    for i, n in enumerate(sizes):
        d += [i] * n
    d += [-1] * (S - len(d))
    d = torch.tensor(d)
    return (d[:, None] == d[None, :]) & (d >= 0)[:, None]


def _masks(B, H, Sq, Skv, g):
    keys = torch.arange(Skv) < torch.tensor([0, 1, 70, Skv])[:B, None]          # the first entry shows nothing at all
    yield "keys", keys[:, None, None, :]
    yield "rows", (torch.rand(Sq, 1, generator=g) < 0.7)
    yield "heads", torch.rand(1, H, Sq, Skv, generator=g) < 0.3
    yield "all", torch.rand(B, H, Sq, Skv, generator=g) < 0.02
    yield "one", torch.rand(Skv, generator=g) < 0.5
    yield "band", ((torch.arange(Sq)[:, None] - torch.arange(Skv)[None, :]).abs() < 20)
    yield "spread", (torch.rand(B, 1, Sq, 2 * Skv, generator=g) < 0.5)[..., ::2]      # keys two bytes apart
    yield "nothing", torch.zeros(1, 1, 1, 1, dtype=torch.bool)


@pytest.mark.parametrize("D,dtype,causal", [(64, BF, False), (128, BF, True), (96, HF, True), (256, HF, False), (256, BF, True)])
def test_boolean_masks(dev, D, dtype, causal):
    B, H, Hkv, Sq, Skv = 4, 4, 2, 200, 331
    q, k, v, do = _draw(B, H, Hkv, Sq, Skv, D, dtype, seed=2)
    for name, mask in _masks(B, H, Sq, Skv, torch.Generator().manual_seed(3)):
        out, lse, grads = _run(dev, q, k, v, do, attn_mask=mask.to(dev), is_causal=causal)
        e = Exact(q, k, v, causal=causal, seen=mask, dout=do)
        _compare(e, out, lse, grads)
        gone = (e.lse == -math.inf).to(dev)
        assert bool((out[gone] == 0).all()) and bool((grads[0][gone] == 0).all()), name


def test_documents_and_wide_masks(dev):
    """Masks whose blocks pass 64 tiles each way, so that whole words of them show nothing."""
    S = 64 * 70 + 5
    mask = _docs(S, (100, 1, 700, 64, 2900))
    q, k, v, do = _draw(1, 2, 1, S, S, 64, BF, seed=8)
    out, lse, grads = _run(dev, q, k, v, do, attn_mask=mask.to(dev))
    _compare(Exact(q, k, v, seen=mask, dout=do), out, lse, grads)
    strip = torch.zeros(S, S, dtype=torch.bool)
    strip[S - 3:, 1] = True
    strip[7, S - 1] = True
    for D in (128, 256):
        q, k, v, do = _draw(1, 1, 1, S, S, D, BF, seed=9)
        out, lse, grads = _run(dev, q, k, v, do, attn_mask=strip.to(dev))
        _compare(Exact(q, k, v, seen=strip, dout=do), out, lse, grads)


def _poison(t, rows, seed=0):
    """Infinities and NaN somewhere in the given rows [.., S, D]."""
    t = t.clone()
    bad = torch.tensor([math.nan, math.inf, -math.inf])
    g = torch.Generator().manual_seed(seed)
    for i, r in enumerate(rows):
        t[:, :, r, int(torch.randint(0, t.shape[-1], (1,), generator=g))] = bad[i % 3].to(t.dtype)
    return t


@pytest.mark.parametrize("D,dtype", [(64, BF), (96, HF), (128, BF), (128, HF), (256, BF)])
def test_what_hidden_places_hold_does_not_matter(dev, D, dtype):
    """Infinities and NaN in keys, values, queries and gradients that nothing sees."""
    B, H, Hkv, S = 2, 2, 1, 300
    q, k, v, do = _draw(B, H, Hkv, S, S, D, dtype, seed=5)
    keys, rows = [3, 64, 65, 130, 299], [0, 70, 201, 298]
    mask = torch.ones(S, S, dtype=torch.bool)
    mask[:, keys] = False
    mask[rows, :] = False
    want = _run(dev, q, k, v, do, attn_mask=mask.to(dev))
    got = _run(dev, _poison(q, rows), _poison(k, keys), _poison(v, keys, 1), _poison(do, rows, 2), attn_mask=mask.to(dev))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for a, b, hidden in zip(want[2], got[2], (rows, keys, keys)):
        assert bool(torch.isfinite(b).all()) and bool((b[:, :, hidden] == 0).all())
        if dtype == BF:      # (fp16's gradients are held times a power of two of the largest rows, which are others now)
            assert torch.equal(a, b)
        else:
            assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -9 * float(a.abs().max())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_a_query_sees_does(dev, D):
    """A query that sees an infinity or a NaN is NaN, the others keep their bits; so with the gradients."""
    B, H, S = 1, 2, 260
    q, k, v, do = _draw(B, H, H, S, S, D, BF, seed=7)
    mask = torch.ones(S, S, dtype=torch.bool).tril()
    want = _run(dev, q, k, v, do, is_causal=True)
    for where in ("q", "k", "v", "do"):
        at = 100
        ts = dict(q=q, k=k, v=v, do=do)
        ts[where] = _poison(ts[where], [at])
        got = _run(dev, ts["q"], ts["k"], ts["v"], ts["do"], is_causal=True)
        rows = torch.zeros(S, dtype=torch.bool)
        rows[at if where in ("q", "do") else slice(at, S)] = True
        nan_out = rows if where != "do" else torch.zeros(S, dtype=torch.bool)
        assert bool(torch.isnan(got[0][:, :, nan_out]).all()) and torch.equal(got[0][:, :, ~nan_out], want[0][:, :, ~nan_out])
        touched = (mask & rows[:, None]).any(0)                    # the keys that such a query sees
        dq, dk, dv = got[2]
        assert bool(torch.isnan(dq[:, :, rows]).any(-1).all()) and torch.equal(dq[:, :, ~rows], want[2][0][:, :, ~rows])
        for a, b in ((dk, want[2][1]), (dv, want[2][2])):
            assert bool(torch.isnan(a[:, :, touched]).any(-1).all()) and torch.equal(a[:, :, ~touched], b[:, :, ~touched])


BIASED = [
    # B, H, Hkv, Sq, Skv, D, dtype, layout, causal, buckets, reach, table type
    (2, 3, 3, 257, 257, 64, BF, "HND", False, 32, 128, BF),
    (2, 4, 2, 200, 333, 128, HF, "NHD", True, 32, 128, torch.float32),
    (1, 2, 1, 1, 300, 64, BF, "HND", True, 16, 40, BF),
    (1, 2, 2, 300, 40, 96, BF, "NHD", False, 8, 20, HF),
    (1, 2, 2, 190, 210, 256, HF, "HND", False, 64, 100, HF),
    (1, 2, 1, 300, 300, 256, BF, "NHD", True, 32, 700, BF),
    (1, 2, 2, 900, 1000, 64, HF, "HND", False, 4, 2, torch.float32),
    (1, 1, 1, 1700, 1700, 64, BF, "HND", False, 256, 760, torch.float32),
]


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D,dtype,layout,causal,buckets,reach,ttype", BIASED)
def test_bias_inside(dev, B, H, Hkv, Sq, Skv, D, dtype, layout, causal, buckets, reach, ttype):
    q, k, v, do = _draw(B, H, Hkv, Sq, Skv, D, dtype, seed=11)
    table = (torch.randn(buckets, H, generator=torch.Generator().manual_seed(12)) * 1.5).to(ttype)
    kw = dict(is_causal=causal, bidirectional=not causal, max_distance=reach)
    out, lse, grads = _run(dev, q, k, v, do, layout, table=table, **kw)
    bucket = bucket_map(Sq, Skv, buckets, reach, not causal)
    bias = table.double()[bucket].permute(2, 0, 1)
    e = Exact(q, k, v, causal=causal, bias=bias, dout=do)
    _compare(e, out, lse, grads[:3])
    side = buckets // 2 if not causal else buckets
    outer = bucket % side == side - 1
    want, room = e.table(bucket, buckets, outer, ttype)
    close(grads[3], want, room)
    again = _run(dev, q, k, v, do, layout, table=table, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, again[2]))
    # the same bias as a tensor: its table's gradient through relative_bias from the same ds
    alone = cdna4_sage.relative_bias(table.to(dev), Sq, Skv, not causal, reach, torch.float32)
    assert torch.equal(alone.double().cpu(), bias)


def test_bias_with_a_mask_and_one_sided_without_causal(dev):
    B, H, Sq, Skv = 2, 2, 150, 220
    q, k, v, do = _draw(B, H, H, Sq, Skv, 64, BF, seed=13)
    g = torch.Generator().manual_seed(14)
    table = torch.randn(32, H, generator=g).to(BF)
    mask = torch.rand(B, 1, Sq, Skv, generator=g) < 0.4
    mask[1, :, 30:60] = False
    bucket = bucket_map(Sq, Skv, 32, 100, False)
    out, lse, grads = _run(dev, q, k, v, do, table=table, attn_mask=mask.to(dev), bidirectional=False, max_distance=100)
    e = Exact(q, k, v, seen=mask, bias=table.double()[bucket].permute(2, 0, 1), dout=do)
    _compare(e, out, lse, grads[:3])
    close(grads[3], *e.table(bucket, 32, bucket == 31, BF))


def test_gradients_are_differences(dev):
    """Along each gradient's own direction the loss moves as the gradient says, up to what the roundings of both allow."""
    H, Sq, Skv, D = 2, 60, 90, 64
    q, k, v, do = _draw(1, H, H, Sq, Skv, D, HF, seed=15)
    table = torch.randn(16, H, generator=torch.Generator().manual_seed(16)).to(HF)
    bucket = bucket_map(Sq, Skv, 16, 30, True)

    def exact(q, k, v, table):
        return Exact(q, k, v, bias=table.double()[bucket].permute(2, 0, 1), dout=do)

    def loss(q, k, v, table):
        out = cdna4_sage.attention_train(*(t.to(dev) for t in (q, k, v)), bias_table=table.to(dev), max_distance=30)
        return float((out.double().cpu() * do.double()).sum())

    _, _, grads = _run(dev, q, k, v, do, table=table, max_distance=30)
    base = [q, k, v, table]
    e = exact(*base)
    rooms = [e.room_dq, e.room_dk, e.room_dv, e.table(bucket, 16, bucket % 8 == 7, HF)[1]]
    exacts = [e.dq, e.dk, e.dv, e.table(bucket, 16, bucket % 8 == 7, HF)[0]]
    for i in range(4):
        way = exacts[i] / exacts[i].abs().max() * 0.25
        plus, minus = list(base), list(base)
        plus[i], minus[i] = (base[i].double() + way).to(HF), (base[i].double() - way).to(HF)
        moved = plus[i].double() - minus[i].double()
        told = float((grads[i].double().cpu() * moved).sum())
        ep, em = exact(*plus), exact(*minus)
        curve = abs(float(((ep.out - em.out) * do.double()).sum()) - float((exacts[i] * moved).sum()))
        noise = float((do.double().abs() * (ep.room_out + em.room_out)).sum()) + float((rooms[i] * moved.abs()).sum())
        assert abs(loss(*plus) - loss(*minus) - told) <= curve + noise
        assert abs(told) > noise, "the step is too small: a gradient of 0 would pass"


@pytest.mark.parametrize("D,dtype,causal,bias", [(64, BF, True, False), (128, BF, False, False), (128, HF, True, True), (256, BF, True, False),
                                                 (96, BF, True, True)])
def test_packed_sequences(dev, D, dtype, causal, bias):
    """Each sequence as a call of its own; empty ones, rows that none covers and q / k offsets of different lengths."""
    H, Hkv = 4, 2
    lq, lk = [0, 5, 130, 1, 300, 64, 0, 17], [3, 5, 200, 0, 300, 65, 0, 128]
    first, more = 7, 9                                     # rows before the first and behind the last sequence
    cu = [torch.tensor([first] + [first + sum(n[:i + 1]) for i in range(len(n))], dtype=torch.int32) for n in (lq, lk)]
    TQ, TK = int(cu[0][-1]) + more, int(cu[1][-1]) + more
    g = torch.Generator().manual_seed(21)
    q, do = (torch.randn(TQ, H, D, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(TK, Hkv, D, generator=g).to(dtype) for _ in range(2))
    for t, c in ((q, cu[0]), (do, cu[0]), (k, cu[1]), (v, cu[1])):
        t[:first], t[int(c[-1]):] = math.nan, math.inf     # (what they hold does not matter)
    table = torch.randn(16, H, generator=g).to(dtype) if bias else None
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)] + ([table.to(dev).requires_grad_()] if bias else [])
    kw = dict(bias_table=leaves[3], max_distance=40, bidirectional=not causal) if bias else {}
    out, lse = cdna4_sage.attention_train_varlen(*leaves[:3], cu[0].to(dev), cu[1].to(dev, torch.int64), is_causal=causal,
                                                 return_lse=True, **kw)
    grads = torch.autograd.grad(out, leaves, do.to(dev))
    assert lse.shape == (H, TQ) and out.shape == q.shape
    total = None
    for b in range(len(lq)):
        rows, keys = slice(int(cu[0][b]), int(cu[0][b + 1])), slice(int(cu[1][b]), int(cu[1][b + 1]))
        one = [t[r].transpose(0, 1)[None] for t, r in ((q, rows), (k, keys), (v, keys), (do, rows))]
        if lq[b] == 0 or lk[b] == 0:
            assert bool((out[rows] == 0).all()) and bool((grads[0][rows] == 0).all())
            assert bool((grads[1][keys] == 0).all()) and bool((grads[2][keys] == 0).all())
            continue
        bucket = bucket_map(lq[b], lk[b], 16, 40, not causal) if bias else None
        e = Exact(*one[:3], causal=causal, dout=one[3], bias=table.double()[bucket].permute(2, 0, 1) if bias else None)
        got = [out[rows], *(t[r] for t, r in zip(grads, (rows, keys, keys)))]
        spread = lambda t: t.transpose(0, 1)[None]  # noqa: E731
        if dtype == HF:      # (the scale of fp16's ds follows from the largest rows of the whole batch)
            e.room_dq, e.room_dk = e.room_dq + 1e-6, e.room_dk + 1e-6
        _compare(e, spread(got[0]), lse[:, rows][None], [spread(t) for t in got[1:]])
        if bias:
            side = 8 if not causal else 16
            w, r = e.table(bucket, 16, bucket % side == side - 1, torch.float32)
            total = (w, r) if total is None else (total[0] + w, total[1] + r)
    if bias:
        close(grads[3], total[0], total[1] + 2.0 ** (-8 if dtype == BF else -11) * total[0].abs())
    for t, c in ((out, cu[0]), (grads[0], cu[0]), (grads[1], cu[1]), (grads[2], cu[1])):
        assert bool((t[:first] == 0).all()) and bool((t[int(c[-1]):] == 0).all())


def test_packed_many_short_sequences_and_bad_offsets(dev):
    """More sequences than a workgroup has threads; offsets that fall or pass the totals give zeros."""
    n, H, D = 700, 2, 64
    lens = [(i * 7) % 5 for i in range(n)]
    cu = torch.tensor([0] + [sum(lens[:i + 1]) for i in range(n)], dtype=torch.int32)
    T = int(cu[-1])
    g = torch.Generator().manual_seed(22)
    q, k, v, do = (torch.randn(T, H, D, generator=g).to(BF) for _ in range(4))
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    out = cdna4_sage.attention_train_varlen(*leaves, cu.to(dev), cu.to(dev), is_causal=True)
    grads = torch.autograd.grad(out, leaves, do.to(dev))
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(lens))
    one = [t.transpose(0, 1)[None] for t in (q, k, v, do)]
    e = Exact(*one[:3], causal=True, seen=seq[:, None] == seq[None, :], dout=one[3])
    for a, want, room in zip((out, *grads), (e.out, e.dq, e.dk, e.dv), (e.room_out, e.room_dq, e.room_dk, e.room_dv)):
        close(a.transpose(0, 1)[None], want, room)
    for bad in (cu.flip(0), cu + 1, cu - 1):
        out = cdna4_sage.attention_train_varlen(*leaves, bad.to(dev), bad.to(dev))
        grads = torch.autograd.grad(out, leaves, do.to(dev))
        assert all(bool((t == 0).all()) for t in (out, *grads))
