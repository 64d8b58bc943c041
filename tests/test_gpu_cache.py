"""The quantized key / value cache: cache_write bit for bit against the definition, cache_read against code * scale,
cache_attention against float64 attention over the same codes, and the step that runs rope, write and attention."""
import math

import pytest
import torch

import cdna4_sage
from cache_util import as_int8, attention, attention_slack, lse_slack, quantize, random_cache, rotate

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _to(dev, cache):
    return cdna4_sage.KVCache(*(t.to(dev) for t in cache))


def _codes_equal(a, b):
    return torch.equal(as_int8(a.cpu()), as_int8(b.cpu()))


def _scales_equal(a, b):
    a, b = a.cpu(), b.cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


# ---- write and read ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("code", [torch.int8, E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_is_the_definition_bit_for_bit(dev, D, code, dtype):
    g = torch.Generator().manual_seed(D)
    tokens, heads, n = 83, 3, 16
    pages = 8
    k = (torch.randn(tokens, heads, D, generator=g) * 10.0 ** torch.randint(-6, 4, (tokens, heads, 1), generator=g)).to(dtype)
    v = torch.randn(tokens, heads, D, generator=g).to(dtype)
    # rows of ties (code + 1/2), zeros, a lone value, the type's ends, infinities and NaN
    k[0] = torch.arange(D).to(dtype) - 3
    k[0, :, 5] = 254
    k[1] = 0
    k[2] = 0
    k[2, :, 7] = -1.5
    k[3] = torch.finfo(dtype).max
    k[4] = torch.finfo(dtype).smallest_normal / 4
    k[5, 0, 1] = float("inf")
    k[5, 1, 2] = float("nan")
    v[6, 2, 3] = float("-inf")
    v[7] = (0.5 ** torch.arange(D).clamp(max=20)).to(dtype)
    slots = torch.randperm(pages * n, generator=g)[:tokens]
    slots[10], slots[11] = -1, pages * n          # tokens without a slot
    cache = cdna4_sage.new_cache(pages, n, heads, D, code, dev)
    as_int8(cache.k).fill_(17)
    cache.k_scale.fill_(3.0)
    cdna4_sage.cache_write(cache, k.to(dev), v.to(dev), slots.to(dev))
    for x, got, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        codes, s = quantize(x, code)
        want, want_s = as_int8(got.cpu()).clone(), scale.cpu().clone()
        if x is k:
            want.fill_(17), want_s.fill_(3.0)
        else:
            want.zero_(), want_s.zero_()
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * n:
                want[slot // n, :, slot % n] = as_int8(codes)[i]
                want_s[slot // n, :, slot % n] = s[i]
        assert _codes_equal(want, got)
        assert _scales_equal(want_s, scale)


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_write_and_read_four_dimensional(dev, layout):
    g = torch.Generator().manual_seed(1)
    B, S, heads, D, n, pages = 3, 21, 5, 128, 32, 7
    fused = torch.randn(B, S, 2 * heads * D, generator=g).to(torch.bfloat16).to(dev)
    k, v = (fused[..., i * heads * D:(i + 1) * heads * D].unflatten(-1, (heads, D)) for i in (0, 1))
    slots = torch.randperm(pages * n, generator=g)[:B * S].view(B, S).to(dev)
    slots[1, 15:] = -1
    a = (k.transpose(1, 2), v.transpose(1, 2)) if layout == "HND" else (k, v)
    cache = cdna4_sage.new_cache(pages, n, heads, D, device=dev)
    cdna4_sage.cache_write(cache, *a, slots, layout)
    packed = cdna4_sage.new_cache(pages, n, heads, D, device=dev)
    cdna4_sage.cache_write(packed, k.reshape(B * S, heads, D), v.reshape(B * S, heads, D), slots.view(-1).int())
    for x, y in zip(cache, packed):
        assert torch.equal(x, y)
    for dtype in (torch.bfloat16, torch.float16):
        rk, rv = cdna4_sage.cache_read(cache, slots, dtype, layout)
        pk, pv = cdna4_sage.cache_read(cache, slots.view(-1).int(), dtype)
        for r, p, x in ((rk, pk, k), (rv, pv, v)):
            r = r.transpose(1, 2) if layout == "HND" else r
            assert r.dtype == dtype and torch.equal(r.reshape(B * S, heads, D), p)
            codes, s = quantize(x.cpu(), torch.int8)
            want = (codes.float() * s.unsqueeze(-1)).to(dtype)
            want[1, 15:] = 0
            assert torch.equal(r.cpu(), want)


@pytest.mark.parametrize("D, heads, tokens", [(64, 5, 53001), (96, 3, 44003), (128, 7, 19001), (256, 3, 22007)])
@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_many_rows_as_in_small_calls(dev, D, heads, tokens, code):
    """Rows of calls that take several per thread, some without a slot at their ends: bit for bit those of small calls."""
    g = torch.Generator().manual_seed(D + heads)
    n, dtype = 64, torch.float16 if D == 96 else torch.bfloat16
    pages = -(-tokens // n) + 1
    k, v = (torch.randn(tokens, heads, D, generator=g).to(dtype).to(dev) for _ in range(2))
    slots = torch.randperm(pages * n, generator=g)[:tokens].to(dev)
    slots[-5:] = torch.tensor([-1, pages * n, int(slots[-3]), -7, 2**40], device=dev)
    one, small = (cdna4_sage.new_cache(pages, n, heads, D, code, dev) for _ in range(2))
    cdna4_sage.cache_write(one, k, v, slots)
    for i in range(0, tokens, 999):
        cdna4_sage.cache_write(small, k[i:i + 999], v[i:i + 999], slots[i:i + 999])
    for x, y in zip(one, small):
        assert torch.equal(as_int8(x) if x.dtype != torch.float32 else x, as_int8(y) if y.dtype != torch.float32 else y)
    codes, scale = quantize(v[-9:].cpu(), code)
    at = int(slots[-3])
    assert _codes_equal(codes[-3], one.v[at // n, :, at % n]) and _scales_equal(scale[-3], one.v_scale[at // n, :, at % n])
    got = cdna4_sage.cache_read(one, slots, dtype)
    for i in range(0, tokens, 999):
        for a, b in zip(got, cdna4_sage.cache_read(small, slots[i:i + 999], dtype)):
            assert torch.equal(a[i:i + 999], b)
    assert not bool(got[0][-2:].any()) and bool(got[0][-3].any())


def test_read_of_every_e4m3_code_and_nan_rows(dev):
    codes = torch.zeros(1, 1, 16, 128, dtype=torch.int8)
    codes[0, 0, :2] = torch.arange(256).to(torch.uint8).view(torch.int8).view(2, 128)
    k = codes.view(E4M3)
    scale = torch.full((1, 1, 16), 0.37)
    scale[0, 0, 3] = float("nan")
    cache = _to(dev, cdna4_sage.KVCache(k, k.clone(), scale, scale.clone()))
    for dtype in (torch.bfloat16, torch.float16):
        got, _ = cdna4_sage.cache_read(cache, torch.arange(4, device=dev), dtype)
        want = (k[0, 0, :4].float() * scale[0, 0, :4, None]).to(dtype)
        assert torch.equal(torch.isnan(got[:, 0].cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got[:, 0].cpu()), torch.nan_to_num(want))


def test_int8_read_of_every_code(dev):
    codes = torch.zeros(1, 1, 16, 256, dtype=torch.int8)
    codes[0, 0, 0] = torch.arange(-128, 128)
    scale = torch.full((1, 1, 16), 0.013)
    cache = _to(dev, cdna4_sage.KVCache(codes, codes.clone(), scale, scale.clone()))
    got, _ = cdna4_sage.cache_read(cache, torch.zeros(1, dtype=torch.int32, device=dev), torch.float16)
    assert torch.equal(got[0, 0].cpu(), (codes[0, 0, 0].float() * scale[0, 0, 0]).half())


def test_write_without_tokens_and_read_of_none(dev):
    cache = cdna4_sage.new_cache(2, 16, 2, 64, device=dev)
    e = torch.empty(0, 2, 64, dtype=torch.float16, device=dev)
    cdna4_sage.cache_write(cache, e, e, torch.empty(0, dtype=torch.int64, device=dev))
    k, v = cdna4_sage.cache_read(cache, torch.empty(0, dtype=torch.int64, device=dev))
    assert k.shape == v.shape == (0, 2, 64)
    assert all(not bool(as_int8(t).any()) if t.dtype != torch.float32 else not bool(t.any()) for t in cache)


# ---- attention --------------------------------------------------------------------------------------------------------

def _table(g, lengths, n, pages, columns=None, fill=-1):
    need = [-(-max(int(x), 0) // n) for x in lengths]
    columns = max(need + [1]) if columns is None else columns
    order = torch.randperm(pages, generator=g).to(torch.int32)
    t = torch.full((len(lengths), columns), fill, dtype=torch.int32)
    at = 0
    for b, x in enumerate(need):
        x = min(x, columns)
        t[b, :x] = order[at:at + x]
        at += x
    assert at <= pages
    return t


def _tree(g, B, T):
    m = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            if i:
                m[b, i] = m[b, int(torch.randint(0, i, (1,), generator=g))]
            m[b, i, i] = True
    return m


def _compare(dev, q, cache, table, lengths, layout="HND", sm_scale=None, is_causal=True, tree=None, on_gpu=None):
    """q [B, H, T, D] on the CPU; on_gpu: the cache the GPU reads where it differs from the reference's."""
    gpu = _to(dev, cache if on_gpu is None else on_gpu)
    qd = (q if layout == "HND" else q.transpose(1, 2).contiguous()).to(dev)
    out, lse = cdna4_sage.cache_attention(qd, gpu, table.to(dev), lengths.to(dev), layout, sm_scale, is_causal,
                                          None if tree is None else tree.to(dev), return_lse=True)
    alone = cdna4_sage.cache_attention(qd, gpu, table.to(dev), lengths.to(dev), layout, sm_scale, is_causal,
                                       None if tree is None else tree.to(dev))
    assert torch.equal(alone, out) and out.shape == qd.shape and out.dtype == q.dtype
    got = (out if layout == "HND" else out.transpose(1, 2)).double().cpu()
    want, want_lse, mag, big = attention(q.double(), cache, table, lengths, sm_scale, is_causal, tree)
    D = q.shape[-1]
    room = attention_slack(mag, big, want, D, q.dtype)
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() / room).max())
    lse = lse.double().cpu()
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), none)
    assert not bool(got[none].any())
    off = torch.where(none, 0.0, (lse - want_lse).abs())
    assert bool((off <= lse_slack(big, torch.where(none, 0.0, want_lse), D)).all()), float(off.max())
    return out


ATTENTION = [
    # T, H, Hkv, D, page, lengths, code, dtype, layout
    (1, 4, 4, 64, 16, [1, 0, 15, 16, 17, 33], torch.int8, torch.float16, "HND"),
    (1, 8, 2, 128, 16, [31, 32, 128, 129, 257], torch.int8, torch.bfloat16, "NHD"),
    (1, 5, 1, 96, 32, [97, 3, 200], E4M3, torch.float16, "HND"),
    (1, 12, 12, 256, 64, [130], E4M3, torch.bfloat16, "HND"),
    (1, 32, 2, 64, 1024, [1500, 9], E4M3, torch.bfloat16, "NHD"),
    (2, 4, 2, 128, 16, [2, 1, 0, 65], torch.int8, torch.float16, "NHD"),
    (5, 8, 2, 96, 16, [5, 40, 300], torch.int8, torch.bfloat16, "HND"),
    (7, 6, 2, 256, 128, [7, 131], torch.int8, torch.float16, "HND"),
    (16, 8, 4, 64, 16, [40, 16, 17], E4M3, torch.bfloat16, "HND"),
    (33, 4, 2, 128, 32, [33, 90, 20], E4M3, torch.float16, "NHD"),
    (70, 2, 1, 64, 16, [70, 101], torch.int8, torch.bfloat16, "HND"),
    (35, 4, 2, 96, 16, [36, 200], torch.int8, torch.float16, "HND"),
    (50, 1, 1, 128, 64, [300, 7], E4M3, torch.bfloat16, "HND"),
    (40, 2, 2, 256, 16, [140, 41], E4M3, torch.float16, "NHD"),
]


@pytest.mark.parametrize("kind", ["causal", "full", "tree"])
@pytest.mark.parametrize("T,H,Hkv,D,page,lengths,code,dtype,layout", ATTENTION)
def test_attention_matches_float64(dev, T, H, Hkv, D, page, lengths, code, dtype, layout, kind):
    g = torch.Generator().manual_seed(T * 1000 + D)
    lengths = torch.tensor(lengths, dtype=torch.int32)
    pages = sum(-(-int(x) // page) for x in lengths) + 2
    cache = random_cache(g, pages, page, Hkv, D, code, spread=0.2)
    table = _table(g, lengths, page, pages)
    q = (torch.randn(len(lengths), H, T, D, generator=g) * 1.5).to(dtype)
    tree = _tree(g, len(lengths), T) if kind == "tree" else None
    _compare(dev, q, cache, table, lengths, layout, is_causal=kind != "full", tree=tree)


@pytest.mark.parametrize("T,H,Hkv", [(1, 8, 1), (9, 6, 2)])
@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_long_sequences_split_over_workgroups(dev, T, H, Hkv, code):
    g = torch.Generator().manual_seed(5)
    lengths = torch.tensor([3001, 517, 0, 128], dtype=torch.int32)
    page, D = 16, 128
    pages = sum(-(-int(x) // page) for x in lengths) + 5
    cache = random_cache(g, pages, page, Hkv, D, code)
    # a table wider than any sequence: its other entries are out of range on both sides
    table = _table(g, lengths, page, pages, columns=400, fill=2**31 - 1)
    table[:, 399] = -2**31
    q = torch.randn(4, H, T, D, generator=g).to(torch.bfloat16)
    _compare(dev, q, cache, table, lengths, tree=_tree(g, 4, T))


@pytest.mark.parametrize("B,T,H,Hkv,D,longest", [
    (70, 1, 8, 4, 64, 500),       # more sequences than lanes, ragged, some empty
    (130, 2, 2, 2, 96, 200),
    (70, 16, 8, 8, 64, 60),       # thousands of rows to join
    (4, 1, 16, 8, 128, 4000),     # sequences in many parts
    (1, 3, 8, 1, 256, 9000),
    (1, 1, 1, 1, 64, 40000),
])
def test_batches_and_splits_of_every_kind(dev, B, T, H, Hkv, D, longest):
    g = torch.Generator().manual_seed(B + longest)
    lengths = torch.randint(0, longest + 1, (B,), generator=g).to(torch.int32)
    lengths[0] = longest
    page = 32
    pages = int(((lengths + page - 1) // page).sum()) + 1
    cache = random_cache(g, pages, page, Hkv, D, torch.int8)
    q = torch.randn(B, H, T, D, generator=g).to(torch.bfloat16)
    _compare(dev, q, cache, _table(g, lengths, page, pages), lengths)


@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_whatever_hidden_places_hold(dev, code):
    """Rows past each length, pages of no sequence, evicted pages and new tokens that no query sees hold NaN scales, NaN
    codes (where no page of the cache is read) and huge scales; the outputs are those of a clean cache."""
    g = torch.Generator().manual_seed(6)
    page, D, Hkv, H, T = 16, 128, 2, 8, 6
    lengths = torch.tensor([37, 6, 90, 3, 0], dtype=torch.int32)
    pages = 20
    cache = random_cache(g, pages, page, Hkv, D, code)
    table = _table(g, lengths, page, pages)
    table[2, 1] = -1                                          # evicted
    table[2, 3] = pages                                       # past the cache
    dirty = [t.clone() for t in cache]
    live = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths.tolist()):
        for j in range(n):
            p = int(table[b, j // page])
            if 0 <= p < pages:
                live[p, j % page] = True
    dead = ~live
    for i, t in enumerate(dirty):
        if i < 2:
            as_int8(t).transpose(1, 2)[dead] = 0x7F           # NaN in E4M3
        else:
            t.transpose(1, 2)[dead] = float("nan") if i == 2 else float("inf")
    tree = _tree(g, len(lengths), T)
    tree[0, :, 4] = False                                     # a drafted token that nobody sees
    at = int(lengths[0]) - T + 4
    for i in (2, 3):
        dirty[i][table[0, at // page], :, at % page] = float("nan")
    tree[1, 3] = False                                        # a row that sees none of the new tokens (and no other)
    q = torch.randn(len(lengths), H, T, D, generator=g).to(torch.float16)
    clean = _compare(dev, q, cache, table, lengths, tree=tree)
    out = _compare(dev, q, cache, table, lengths, tree=tree, on_gpu=dirty)
    assert torch.equal(out, clean)


def test_nan_keys_reach_only_the_rows_that_see_them(dev):
    g = torch.Generator().manual_seed(7)
    page, D, Hkv, H, T = 16, 64, 2, 4, 5
    cache = list(random_cache(g, 8, page, Hkv, D, torch.int8))
    table = torch.arange(8, dtype=torch.int32).view(2, 4)
    lengths = torch.tensor([40, 33], dtype=torch.int32)
    bad = 38                                                   # sequence 0's new token 3
    cache[3][bad // page, 1, bad % page] = float("nan")
    q = torch.randn(2, H, T, D, generator=g).to(torch.bfloat16)
    out = cdna4_sage.cache_attention(q.to(dev), _to(dev, cache), table.to(dev), lengths.to(dev)).cpu()
    nan = torch.isnan(out).any(-1)
    want = torch.zeros(2, H, T, dtype=torch.bool)
    want[0, 2:, 3:] = True                                     # kv head 1, the rows from token 3 on
    assert torch.equal(nan, want)
    q[1, 3, 2, 9] = float("inf")
    out = cdna4_sage.cache_attention(q.to(dev), _to(dev, random_cache(g, 8, page, Hkv, D, torch.int8)), table.to(dev),
                                     lengths.to(dev)).cpu()
    nan = ~torch.isfinite(out).all(-1)
    want.zero_()
    want[1, 3, 2] = True
    assert torch.equal(nan, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_very_different_magnitudes(dev, dtype):
    """Values whose scales span 10^12, zero rows and keys that dominate: the weights keep their bits; queries near the
    ends of bfloat16's range too."""
    g = torch.Generator().manual_seed(8)
    page, D, Hkv, H = 16, 128, 2, 4
    cache = list(random_cache(g, 24, page, Hkv, D, torch.int8))
    cache[3] *= 10.0 ** (-12.0 * torch.rand(cache[3].shape, generator=g))
    cache[3][::3] = 0.0
    lengths = torch.tensor([300, 70], dtype=torch.int32)
    table = _table(g, lengths, page, 24)
    q = torch.randn(2, H, 3, D, generator=g)
    _compare(dev, q.to(dtype), cache, table, lengths)
    if dtype == torch.bfloat16:
        cache[2] = cache[2] * 2.0**-100
        _compare(dev, (q * 2.0**100).to(dtype), cache, table, lengths)
        cache[2] = cache[2] * 2.0**110
        _compare(dev, (q * 2.0**-10).to(dtype), cache, table, lengths)
    cache[3].zero_()
    _compare(dev, q.to(dtype), cache, table, lengths)


@pytest.mark.parametrize("kind", ["causal", "full", "tree"])
@pytest.mark.parametrize("T, H, Hkv, D, code, dtype", [(33, 8, 2, 128, torch.int8, torch.bfloat16), (35, 4, 1, 128, E4M3, torch.float16),
                                                       (45, 6, 2, 96, torch.int8, torch.float16), (29, 5, 1, 96, E4M3, torch.bfloat16),
                                                       (27, 5, 1, 96, E4M3, torch.bfloat16)])
def test_wide_tables(dev, T, H, Hkv, D, code, dtype, kind):
    """Tables of far more columns than the lengths use, whose width alone makes the largest blocks of rows."""
    g = torch.Generator().manual_seed(T)
    lengths = torch.tensor([T + 400, T, 0, T - 7, 1300], dtype=torch.int32)
    page = 64
    pages = sum(-(-max(int(x), 0) // page) for x in lengths) + 2
    cache = random_cache(g, pages, page, Hkv, D, code, spread=0.2)
    q = torch.randn(5, H, T, D, generator=g).to(dtype)
    table = _table(g, lengths, page, pages, columns=2500)
    tree = _tree(g, 5, T) if kind == "tree" else None
    _compare(dev, q, cache, table, lengths, is_causal=kind != "full", tree=tree)
    holes = table.clone()
    holes[0, 2] = -1
    _compare(dev, q, cache, holes, lengths, is_causal=kind != "full", tree=tree)


@pytest.mark.parametrize("T, H, Hkv, D, code", [(150, 3, 1, 128, torch.int8), (301, 1, 1, 64, E4M3), (97, 4, 2, 256, torch.int8)])
def test_prompts_of_many_row_blocks(dev, T, H, Hkv, D, code):
    """Prompts whose earlier rows end before the later ones' keys begin, one behind a prefix, one longer than its keys."""
    g = torch.Generator().manual_seed(T)
    lengths = torch.tensor([T, T + 333, T - 40], dtype=torch.int32)
    page = 16
    pages = sum(-(-int(x) // page) for x in lengths) + 1
    cache = random_cache(g, pages, page, Hkv, D, code, spread=0.2)
    q = torch.randn(3, H, T, D, generator=g).to(torch.bfloat16)
    table = _table(g, lengths, page, pages)
    _compare(dev, q, cache, table, lengths)
    _compare(dev, q, cache, table, lengths, is_causal=False)


@pytest.mark.parametrize("rows", [3, 20, 44])
@pytest.mark.parametrize("score, value, zeros", [(1, 1, 0), (1, -1, 0), (-1, 1, 0), (-1, -1, 0), (1, 0, 300), (-1, 0, 300), (0, 1, 520),
                                                 (0, -1, 40)])
def test_scores_and_values_that_change_along_the_sequence(dev, rows, score, value, zeros):
    """Scores that rise or fall by some hundreds and values that grow or shrink by 2^160 along the keys, values of 0 first
    (rows whose sum is all from them for a while): the running reference follows and loses no weight that counts."""
    g = torch.Generator().manual_seed(rows)
    page, D, n = 16, 128, 610
    cache = list(random_cache(g, 40, page, 1, D, torch.int8))
    lengths = torch.tensor([n], dtype=torch.int32)
    table = torch.arange(40, dtype=torch.int32)[None]
    at = torch.arange(640).view(40, 1, page) / 640
    q = torch.randn(1, rows, 1, D, generator=g).abs() * 4
    if score:
        cache[0] = torch.sign(torch.randn(1, 1, 1, D, generator=g)).expand(40, 1, page, D).to(torch.int8) * 40 + cache[0] // 16
        cache[2] = cache[2] * 0 + 0.04 * (at if score > 0 else 1 - at)
    if value:
        cache[3] = cache[3] * 2.0 ** (160 * value * (at - 0.5))
    cache[3].view(-1)[:zeros] = 0
    _compare(dev, q.to(torch.bfloat16), cache, table, lengths)
    _compare(dev, -q.to(torch.bfloat16), cache, table, lengths, sm_scale=0.7)


def test_scales_masks_and_tables_in_other_forms(dev):
    g = torch.Generator().manual_seed(9)
    page, D, Hkv, H, T = 32, 64, 2, 6, 4
    lengths = torch.tensor([50, 64, 4], dtype=torch.int64)
    cache = random_cache(g, 9, page, Hkv, D, E4M3)
    table = _table(g, lengths, page, 9, columns=3)
    q = torch.randn(3, H, T, D, generator=g).to(torch.bfloat16)
    a = _compare(dev, q, cache, table, lengths, sm_scale=0.31)
    wide = torch.full((3, 7), 5, dtype=torch.int64)
    wide[:, 1:7:2] = table
    qd, gpu, ld = q.to(dev), _to(dev, cache), lengths.to(dev)
    strided = torch.empty(H, 3, T, D + 8, dtype=q.dtype, device=dev).transpose(0, 1)[..., :D].copy_(qd)
    for t in (table.long().to(dev), wide.to(dev)[:, 1:7:2], wide.int().to(dev)[:, 1:7:2]):
        assert torch.equal(cdna4_sage.cache_attention(strided, gpu, t, ld, sm_scale=0.31), a)
    one = _tree(g, 1, T)
    per = cdna4_sage.cache_attention(qd, gpu, table.to(dev), ld, tree_mask=one.expand(3, T, T).contiguous().to(dev))
    for m in (one[0], one, one.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(cdna4_sage.cache_attention(qd, gpu, table.to(dev), ld, tree_mask=m.to(dev)), per)
    low = torch.ones(T, T, dtype=torch.bool).tril()
    assert torch.equal(cdna4_sage.cache_attention(qd, gpu, table.to(dev), ld, tree_mask=low.to(dev)),
                       cdna4_sage.cache_attention(qd, gpu, table.to(dev), ld))
    # lengths past the table are its capacity, negative ones 0
    big = torch.tensor([2**31 - 1, 96, -7], dtype=torch.int32)
    table[:, :] = torch.arange(9).view(3, 3)
    _compare(dev, q, cache, table, big)


def test_refusals(dev):
    cache = cdna4_sage.new_cache(4, 16, 2, 64, device=dev)
    q = torch.zeros(2, 4, 3, 64, dtype=torch.float16, device=dev)
    table, lengths = torch.zeros(2, 2, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    tree = torch.ones(3, 3, dtype=torch.bool, device=dev)
    ok = dict(q=q, cache=cache, block_table=table, lengths=lengths, tensor_layout="HND", sm_scale=None, is_causal=True,
              tree_mask=None)
    cdna4_sage.cache_attention(**ok)
    wide = cdna4_sage.new_cache(4, 16, 2, 128, device=dev)
    bad = [dict(q=q.float()), dict(q=q[0]), dict(q=q.cpu()), dict(q=q[:, :3]), dict(cache=wide), dict(tensor_layout="x"),
           dict(block_table=table[:1]), dict(block_table=table.float()), dict(block_table=table.cpu()), dict(block_table=table[0]),
           dict(lengths=lengths[:1]), dict(lengths=lengths.float()), dict(lengths=lengths.cpu()),
           dict(lengths=lengths.view(2, 1)), dict(tree_mask=tree.int()), dict(tree_mask=tree[:2]), dict(tree_mask=tree.cpu()),
           dict(tree_mask=tree.expand(3, 3, 3)), dict(tree_mask=tree, is_causal=False),
           dict(block_table=table[:, :1].expand(2, 2**26 + 1)),    # more keys than the kernel counts
           dict(cache=cache._replace(v=cache.v.cpu())), dict(cache=cache._replace(k=cache.k.transpose(0, 1)))]
    for kw in bad:
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.cache_attention(**{**ok, **kw})
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for k, v, s in ((x, x, slots[:2]), (x, x, slots.float()), (x, x, slots.cpu()), (x, x.cpu(), slots), (x[:, :1], x[:, :1], slots),
                    (x.view(1, 3, 2, 64), x.view(1, 3, 2, 64), slots), (x[..., :32], x[..., :32], slots)):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.cache_write(cache, k, v, s, "NHD")
    for s in (slots.float(), slots.cpu(), slots.view(1, 1, 3)):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.cache_read(cache, s)
    assert not bool(cache.k_scale.any())


def test_no_queries_and_no_keys(dev):
    cache = cdna4_sage.new_cache(2, 16, 2, 64, device=dev)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn(0, 4, 1, 64, device=dev).half()
    assert cdna4_sage.cache_attention(q, cache, z(0, 2), z(0)).shape == q.shape
    q = torch.randn(2, 4, 0, 64, device=dev).half()
    assert cdna4_sage.cache_attention(q, cache, z(2, 2), z(2)).shape == q.shape
    q = torch.randn(2, 4, 3, 64, device=dev).half()
    out, lse = cdna4_sage.cache_attention(q, cache, z(2, 0), z(2), return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    out, lse = cdna4_sage.cache_attention(q, cache, z(2, 2), z(2), return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())


def test_workspace(dev):
    from cdna4_sage import _capi

    sizes = lambda D, n: _capi.cache_attn_workspace(1, 8, 2, 1, D, 256, n)  # noqa: E731
    assert _capi.cache_attn_workspace(1, 8, 2, 1, 64, 16, 1) == 0               # one step of keys: nothing to join
    assert all(sizes(D, 64) > 0 for D in (64, 96, 128, 256))
    P, n = 0x10000, sizes(64, 64)
    ok = dict(q=P, qsb=512, qss=512, qsh=64, out=P, osb=512, oss=512, osh=64, lse=None, k8=P, ks=P, v8=P, vs=P, table=P,
              ts=4, lengths=P, tree=None, msb=0, msq=0, msk=0, B=1, H=8, Hkv=2, T=1, D=64, dtype=0, ct=0, pages=4, n=256,
              max_pages=64, causal=1, sm=0.0, ws=P, wsb=n, stream=None)
    for bad in (dict(ws=None), dict(wsb=n - 1), dict(ws=P + 64)):   # refused before anything is launched
        with pytest.raises(_capi.SageError, match="workspace"):
            _capi.call("sage_cache_attn", *{**ok, **bad}.values())


def test_cache_beyond_32_bit_offsets(dev):
    """Codes past 4 GiB: the last pages of a cache of 2 x 4.5 GiB hold a copy of the first ones' rows."""
    page, D, Hkv, H = 256, 128, 8, 16
    pages = (9 << 29) // (page * D * Hkv) + 3
    cache = cdna4_sage.new_cache(pages, page, Hkv, D, device=dev)
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randn(300, Hkv, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    near = torch.arange(300, device=dev)
    far = near + (pages - 2) * page
    assert int(far[0]) * Hkv * D > 2**32
    cdna4_sage.cache_write(cache, k, v, near)
    cdna4_sage.cache_write(cache, k, v, far)
    for a, b in zip(cdna4_sage.cache_read(cache, near), cdna4_sage.cache_read(cache, far)):
        assert torch.equal(a, b)
    q = torch.randn(1, H, 1, D, generator=g).to(torch.bfloat16).to(dev)
    length = torch.tensor([300], dtype=torch.int32, device=dev)
    a, b = (cdna4_sage.cache_attention(q, cache, torch.tensor([[p, p + 1]], dtype=torch.int32, device=dev), length)
            for p in (0, pages - 2))
    assert torch.equal(a, b) and bool(a.any())


# ---- the step, streams, graphs, tracing -------------------------------------------------------------------------------

def _decode(dev, code, dtype, layout="NHD", D=128, interleaved=False):
    """A prompt and four steps (the last a tree) through rope, write and attention, against float64 attention over the
    codes that the write is defined to keep."""
    g = torch.Generator().manual_seed(11)
    B, H, Hkv, n, columns = 2, 8, 2, 16, 8
    pages = B * columns
    cache = cdna4_sage.new_cache(pages, n, Hkv, D, code, dev)
    table = torch.randperm(pages, generator=g).to(torch.int32).view(B, columns).to(dev)
    freqs, factor = cdna4_sage.rope_frequencies(D // 2, device=dev)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    kept = None
    for turn, T in enumerate((37, 1, 1, 3, 6)):
        lengths = lengths + T
        q, k, v = (torch.randn(B, T, h, D, generator=g).to(dtype).to(dev) for h in (H, Hkv, Hkv))
        slots = cdna4_sage.cache_slots(table, lengths, T, n)
        tree = _tree(g, B, T).to(dev) if turn == 4 else None
        ts = [t.transpose(1, 2) if layout == "HND" else t for t in (q, k, v)]
        out = cdna4_sage.cache_step(*ts, cache, slots, table, lengths, freqs=freqs, tensor_layout=layout,
                                    interleaved=interleaved, factor=factor, tree_mask=tree)
        out = out.transpose(1, 2) if layout == "HND" else out
        pos = lengths[:, None] - T + torch.arange(T, device=dev)
        rq, rk = cdna4_sage.rope(q, k, pos, freqs, "NHD", interleaved, factor)
        turned, _ = rotate(q.double().cpu(), pos.cpu(), freqs.cpu(), interleaved, factor)
        assert float((rq.double().cpu() - turned).abs().max()) <= 0.05
        kc, ksc = quantize(rk.cpu(), code)
        vc, vsc = quantize(v.cpu(), code)
        if kept is None:
            kept = [torch.zeros_like(t.cpu()) for t in cache]
        page, row = slots.cpu() // n, slots.cpu() % n
        for t, x in zip(kept, (kc, vc, ksc, vsc)):
            (as_int8(t) if t.dim() == 4 else t)[page, :, row] = as_int8(x) if t.dim() == 4 else x
        for a, b in zip(cache, kept):
            assert torch.equal(as_int8(a.cpu()) if a.dim() == 4 else a.cpu(), as_int8(b) if b.dim() == 4 else b)
        want, _, mag, big = attention(rq.transpose(1, 2).double().cpu(), kept, table.cpu(), lengths.cpu(),
                                      tree=None if tree is None else tree.cpu())
        room = attention_slack(mag, big, want, D, dtype)
        off = (out.transpose(1, 2).double().cpu() - want).abs()
        assert bool((off <= room).all()), (turn, float((off / room).max()))


@pytest.mark.parametrize("code,dtype,layout,D,interleaved", [
    (torch.int8, torch.bfloat16, "NHD", 128, False), (E4M3, torch.float16, "HND", 64, True),
    (torch.int8, torch.float16, "HND", 96, True), (E4M3, torch.bfloat16, "NHD", 256, False)])
def test_decoding_loop(dev, code, dtype, layout, D, interleaved):
    _decode(dev, code, dtype, layout, D, interleaved)


def test_prefix_read_back_feeds_the_dense_attention(dev):
    """A prompt chunk over a cached prefix: cache_read gives sageattn its K and V; cache_attention of the same rows agrees
    within what the dense path's own quantization allows (cosine, as its tests have it)."""
    import sageattention

    g = torch.Generator().manual_seed(12)
    H, Hkv, D, n, length, T = 16, 4, 128, 64, 2100, 700
    pages = -(-length // n)
    cache = cdna4_sage.new_cache(pages, n, Hkv, D, device=dev)
    k, v = (torch.randn(length, Hkv, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    slots = torch.arange(length, device=dev)
    cdna4_sage.cache_write(cache, k, v, slots)
    q = torch.randn(1, T, H, D, generator=g).to(torch.bfloat16).to(dev)
    rk, rv = (t.unsqueeze(0) for t in cdna4_sage.cache_read(cache, slots))
    dense = sageattention.sageattn(q, rk, rv, tensor_layout="NHD", is_causal=True)
    own = cdna4_sage.cache_attention(q, cache, torch.arange(pages, dtype=torch.int32, device=dev).view(1, -1),
                                     torch.tensor([length], dtype=torch.int32, device=dev), "NHD")
    a, b = dense.double().flatten(), own.double().flatten()
    assert float(a @ b / (a.norm() * b.norm())) >= 0.999


def test_streams_and_graph(dev):
    g = torch.Generator().manual_seed(13)
    B, T, H, Hkv, D, n = 3, 2, 8, 2, 128, 16
    lengths = torch.tensor([700, 33, 2], dtype=torch.int32, device=dev)
    cache = _to(dev, random_cache(g, 60, n, Hkv, D, torch.int8))
    table = torch.stack([torch.arange(i * 20, i * 20 + 20) for i in range(3)]).to(torch.int32)
    table = torch.cat([table, torch.full((3, 40), -1, dtype=torch.int32)], 1)
    table[0, :44] = torch.arange(16, 60)
    table = table.to(dev)
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(torch.bfloat16).to(dev) for h in (H, Hkv, Hkv))
    freqs = cdna4_sage.rope_frequencies(D)[0].to(dev)

    def step_of(q, cache):
        slots = cdna4_sage.cache_slots(table, lengths, T, n)
        return cdna4_sage.cache_step(q, k, v, cache, slots, table, lengths, freqs=freqs, tensor_layout="NHD")

    copy = lambda: cdna4_sage.KVCache(*(t.clone() for t in cache))  # noqa: E731
    eager = step_of(q, copy())
    c2 = copy()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step_of(q, c2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, eager)
    torch.cuda.synchronize()
    # two graphs of the same calls, each on a cache of its own, replayed in turn, with eager calls between
    graphs = []
    for _ in range(2):
        c = copy()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step_of(q, c)
        graphs.append((graph, out, c))
    ce = copy()
    for i in range(4):
        noise = torch.randn(1 << 18, device=dev).sum()
        want = step_of(q, ce)
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, _ in graphs:
            assert torch.equal(out, want), i
        assert torch.isfinite(noise)
        lengths += torch.tensor([1, 3, 1], dtype=torch.int32, device=dev)   # the graphs read the lengths on the device


def test_threads_on_streams_of_their_own(dev):
    """Calls of several sizes at once, from threads with a stream each: every one gives what it gives alone."""
    import threading

    g = torch.Generator().manual_seed(21)
    page, D, Hkv = 16, 64, 2
    cache = _to(dev, random_cache(g, 200, page, Hkv, D, E4M3))
    freqs = cdna4_sage.rope_frequencies(D)[0].to(dev)

    def job(i):
        gi = torch.Generator().manual_seed(i)
        lengths = torch.randint(1, 700, (3 + i,), generator=gi, dtype=torch.int32)
        table = torch.randint(0, 200, (3 + i, 44), generator=gi, dtype=torch.int32).to(dev)
        q = torch.randn(3 + i, 4, 1 + 3 * i, D, generator=gi).to(torch.bfloat16).to(dev)
        lengths = lengths.to(dev)

        def run():
            x = cdna4_sage.rope(q, None, None, freqs)
            return cdna4_sage.cache_attention(x, cache, table, lengths, return_lse=True)

        return run

    jobs = [job(i) for i in range(4)]
    want = [run() for run in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(15):
                got = jobs[i]()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_traced(dev):
    g = torch.Generator().manual_seed(14)
    B, T, H, Hkv, D, n = 2, 3, 4, 2, 64, 16
    lengths = torch.tensor([20, 9], dtype=torch.int32, device=dev)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    base = _to(dev, random_cache(g, 4, n, Hkv, D, E4M3))
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(torch.bfloat16).to(dev) for h in (H, Hkv, Hkv))
    slots = cdna4_sage.cache_slots(table, lengths, T, n)

    def fn(q, k, v, k8, v8, ks, vs):
        cache = cdna4_sage.KVCache(k8, v8, ks, vs)
        cdna4_sage.cache_write(cache, k, v, slots, "NHD")
        out, lse = cdna4_sage.cache_attention(q, cache, table, lengths, "NHD", return_lse=True)
        return (out, lse, cdna4_sage.cache_attention(q, cache, table, lengths, "NHD", is_causal=False),
                *cdna4_sage.cache_read(cache, slots, torch.float16, "HND"))

    c1, c2 = (tuple(t.clone() for t in base) for _ in range(2))
    want = fn(q, k, v, *c1)
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(q, k, v, *c2)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for a, b in zip(c1, c2):
        assert torch.equal(as_int8(a) if a.dim() == 4 else a, as_int8(b) if b.dim() == 4 else b)
    qg = q.clone().requires_grad_(True)                        # no derivative: the backward raises
    out = cdna4_sage.cache_attention(qg, base, table, lengths, "NHD")
    with pytest.raises(RuntimeError):
        out.sum().backward()
