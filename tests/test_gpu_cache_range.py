"""cache_attention at the ends of its range: tiny and infinite queries, values of very different sizes side by side, places
that a row does not see, and the joining of many rows that come in several parts each."""
import math

import pytest
import torch

import cdna4_sage
from cache_util import attention, random_cache, score_slack
from cdna4_sage import _capi
from test_gpu_cache import _compare, _table, _to, _tree

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("rows", [3, 20, 44])
@pytest.mark.parametrize("power, sm_scale", [(-112, None), (-120, None), (-131, None), (-100, 2.0**-30), (-112, 2.0**-20),
                                             (10, 2.0**-126)])
def test_small_queries_and_scales_beside_large_keys(dev, rows, power, sm_scale):
    """Scores that are far from both ends of float32's range, of factors that are not: keys of 2^99, queries and scales down
    to the smallest."""
    g = torch.Generator().manual_seed(rows)
    page, D, n = 16, 256, 70
    cache = list(random_cache(g, 5, page, 1, D, torch.int8))
    sign = torch.sign(torch.randn(D, generator=g))
    cache[0] = (sign * torch.randint(60, 128, (5, 1, page, D), generator=g)).to(torch.int8)
    cache[2] = 2.0 ** (92.0 * torch.rand(5, 1, page, generator=g).sqrt())
    cache[2][-1] = 2.0**92
    q = (sign * torch.rand(1, rows, 1, D, generator=g) * 2.0**power).to(torch.bfloat16)
    assert bool(q.any())
    lengths = torch.tensor([n], dtype=torch.int32)
    _compare(dev, q, cache, torch.arange(5, dtype=torch.int32)[None], lengths, sm_scale=sm_scale)


@pytest.mark.parametrize("rows, D", [(1, 64), (2, 128), (24, 96), (20, 256), (44, 128)])
@pytest.mark.parametrize("high", [0, 1, 2, 3])
def test_neighbouring_tiles_of_very_different_values(dev, rows, D, high):
    """One tile of 32 keys in four has values of 2^93, the others of 2^-86, with scores alike: each wave has a reference of its
    own, 2^179 apart, and the sums have to come together all the same."""
    g = torch.Generator().manual_seed(rows + high)
    page, n = 32, 256 - 7
    cache = list(random_cache(g, 8, page, 1, D, torch.int8))
    tile = torch.arange(8).view(8, 1, 1) % 4
    cache[3] = torch.where(tile == high, 2.0**86, 2.0**-93) * (1 + torch.rand(8, 1, page, generator=g))
    q = torch.randn(1, rows, 1, D, generator=g).to(torch.bfloat16)
    table, lengths = torch.arange(8, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    _compare(dev, q, cache, table, lengths)
    cache[3] = torch.where(tile == high, 2.0**-93, 2.0**86) * (1 + torch.rand(8, 1, page, generator=g))
    _compare(dev, q, cache, table, lengths)


@pytest.mark.parametrize("rows, D", [(1, 64), (3, 128), (20, 128), (44, 128), (44, 96), (20, 256)])
@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_a_row_never_changes_with_what_it_does_not_see(dev, rows, D, code):
    """Weights whose largest lies within a factor of two of where the running reference is raised, beside scales of hidden
    keys, and beside other rows, that are far above: the bits stay."""
    page, n = 16, 150
    differ = 0
    for seed in range(12):
        g = torch.Generator().manual_seed(100 * seed + rows)
        cache = list(random_cache(g, 10, page, 1, D, code))
        codes = cache[0].float()
        codes.view(160, D)[:] = torch.randint(-2, 3, (160, D), generator=g)
        codes.view(160, D)[140] = 96
        cache[0] = codes.to(code)
        q = (0.5 + torch.rand(1, rows, 1, D, generator=g)).to(torch.float16)
        # the score of key 140 is 7.6 to 8.3 in units of ln 2, those of the others next to 0
        cache[2] = cache[2] * 0 + 2.0**-12
        cache[2].view(-1)[140] = (7.6 + seed / 16) * math.log(2) / (96 * D) * D**0.5
        table, lengths = torch.arange(10, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
        run = lambda q, c, l=lengths, **kw: cdna4_sage.cache_attention(  # noqa: E731
            q.to(dev), _to(dev, c), table.to(dev), l.to(dev), return_lse=True, **kw)
        clean = run(q, cache)
        for value in (math.inf, 1e30, 1e4):
            dirty = [t.clone() for t in cache]
            dirty[3].view(-1)[n:] = value
            for a, b in zip(clean, run(q, dirty)):
                differ += not torch.equal(a, b)
        # the last row alone changes: queries of other rows do not reach the first ones
        if rows > 1:
            other = q.clone()
            other[0, -1] *= 30
            for a, b in zip(clean, run(other, cache)):
                differ += not torch.equal(a[:, :-1], b[:, :-1])
        # what comes behind a new token: the first of two new tokens beside a second of other sizes
        two = torch.cat([q, q], 2)
        late = [t.clone() for t in cache]
        late[3].view(-1)[n - 1] = 1e20
        for a, b in zip(run(two, cache), run(two, late)):
            differ += not torch.equal(a[:, :, 0], b[:, :, 0])
    assert differ == 0


@pytest.mark.parametrize("T, H, Hkv, D", [(1, 4, 2, 64), (3, 10, 1, 128), (7, 7, 1, 96), (5, 8, 2, 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_an_infinite_query_gives_nan_where_it_sees_a_key(dev, T, H, Hkv, D, dtype, sign, code):
    """The infinite channel meets codes of one sign only, or none but zeros: scores of -inf, +inf or NaN alone."""
    g = torch.Generator().manual_seed(T)
    lengths = torch.tensor([90, T, max(T - 2, 0), 0], dtype=torch.int32)
    page, pages = 16, 16
    cache = list(random_cache(g, pages, page, Hkv, D, code))
    c = int(torch.randint(0, D, (1,), generator=g))
    k = cache[0].float()
    k[..., c] = sign * k[..., c].abs().clamp(min=1)
    k[..., (c + 1) % D] = 0
    cache[0] = k.to(code)
    table = _table(g, lengths, page, pages)
    q = torch.randn(4, H, T, D, generator=g).to(dtype)
    clean = cdna4_sage.cache_attention(q.to(dev), _to(dev, cache), table.to(dev), lengths.to(dev), return_lse=True)
    bad = torch.zeros(4, H, T, dtype=torch.bool)
    bad[:, 0, T - 1], bad[:, H - 1, 0], bad[:, H // 2, T // 2] = True, True, True
    for at, value in ((c, -math.inf), (c, math.inf), ((c + 1) % D, math.inf), (c, math.nan)):
        x = q.clone()
        x[..., at][bad] = value
        out, lse = cdna4_sage.cache_attention(x.to(dev), _to(dev, cache), table.to(dev), lengths.to(dev), return_lse=True)
        sees = torch.zeros(4, H, T, dtype=torch.bool)
        for b, n in enumerate(lengths.tolist()):
            sees[b, :, max(T - n, 0):] = True
        want = bad & sees
        assert torch.equal(torch.isnan(out.cpu()).all(-1), want) and torch.equal(torch.isnan(out.cpu()).any(-1), want)
        assert torch.equal(torch.isnan(lse.cpu()), want)
        assert not bool(out.cpu()[~sees].any()) and bool((lse.cpu()[~sees] == -math.inf).all())
        for a, b in zip((out.cpu(), lse.cpu()), clean):
            assert torch.equal(a[~want], b.cpu()[~want])


def _parts(lengths, workers):
    """Ranges that each sequence's steps (128 keys, one at least) lie in, cut evenly as the kernel's header says."""
    steps = [max(-(-int(n) // 128), 1) for n in lengths]
    total = sum(steps)
    workers = min(workers, total)
    per, longer = divmod(total, workers)
    of = lambda s: s // (per + 1) if s < longer * (per + 1) else longer + (s - longer * (per + 1)) // per  # noqa: E731
    out, at = [], 0
    for s in steps:
        out.append(of(at + s - 1) - of(at) + 1)
        at += s
    return out


@pytest.mark.parametrize("D, T, H, Hkv, B, long, columns, rt, code, dtype", [
    (128, 35, 6, 2, 41, 4000, 125, 2, torch.int8, torch.bfloat16),
    (128, 35, 6, 2, 41, 4000, 940, 3, torch.int8, torch.float16),
    (96, 21, 5, 1, 83, 3000, 94, 2, E4M3, torch.float16),
    (96, 21, 10, 2, 43, 3000, 1500, 3, E4M3, torch.bfloat16),
    (256, 13, 6, 2, 107, 3500, 112, 2, torch.int8, torch.bfloat16),
    (64, 27, 6, 2, 53, 3500, 120, 2, E4M3, torch.float16),
    (128, 1, 32, 4, 270, 6000, 200, 1, torch.int8, torch.bfloat16),
])
@pytest.mark.parametrize("kind", ["causal", "tree"])
def test_many_rows_in_several_parts(dev, D, T, H, Hkv, B, long, columns, rt, code, dtype, kind):
    """More than 8192 rows to join, of sequences in 1, 2 to 4 and more than 4 parts; groups of four rows that cross blocks of
    rows, and last ones of fewer."""
    g = torch.Generator().manual_seed(D + T)
    page = 32
    lengths = torch.randint(max(T - 3, 0), 700, (B,), generator=g).to(torch.int32)
    lengths[B // 3] = long
    lengths[B // 2] = 0
    rows = T * (H // Hkv)
    assert rows * B * Hkv > 8192
    part_rows = min(rows, 16 * rt)
    unit = Hkv * -(-rows // (16 * rt)) * 2 * part_rows
    # the plan's ranges from its workspace: [unit][ranges] rows of D + 1 floats
    workers = _capi.cache_attn_workspace(B, H, Hkv, T, D, page, columns) // (4 * (D + 1) * unit)
    parts = _parts(lengths, workers)
    assert 8 < workers <= 4 * B and max(parts) > 4 and any(2 <= p <= 4 for p in parts), (workers, sorted(set(parts)))
    pages = sum(-(-int(x) // page) for x in lengths) + 1
    cache = random_cache(g, pages, page, Hkv, D, code, spread=0.2)
    q = torch.randn(B, H, T, D, generator=g).to(dtype)
    table = _table(g, lengths, page, pages, columns=columns)
    _compare(dev, q, cache, table, lengths, "NHD" if kind == "tree" else "HND", tree=_tree(g, B, T) if kind == "tree" else None)


@pytest.mark.parametrize("T, H, Hkv, D, n, code", [(1, 8, 1, 64, 100, torch.int8), (1, 16, 2, 128, 300, E4M3), (4, 12, 3, 96, 120, torch.int8),
                                                   (1, 16, 1, 256, 90, torch.int8), (16, 2, 2, 64, 1500, E4M3)])
def test_weights_of_few_rows_keep_their_bits(dev, T, H, Hkv, D, n, code):
    """Up to 16 rows per kv head: two float16 numbers per weight, each rounded to the nearest (2^-11 and 2^-11 of the rest: 2^-22),
    where one would leave 2^-11.  Scores are small, so products lie within 2^-9 of the largest, which is at 2^6 or more: the second
    number's own steps, 2^-24, are below 2^-22 of the product too."""
    g = torch.Generator().manual_seed(n)
    page = 32
    pages = -(-n // page)
    cache = random_cache(g, pages, page, Hkv, D, code)
    q = (torch.randn(1, H, T, D, generator=g) / 64).to(torch.float16)
    table, lengths = torch.arange(pages, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    want, _, mag, big = attention(q.double(), cache, table, lengths)
    got = cdna4_sage.cache_attention(q.to(dev), _to(dev, cache), table.to(dev), lengths.to(dev)).double().cpu()
    # (the float32 sums and exponentials: 2^-20, as attention_slack has it)
    room = mag * (2.0**-22 + 2.0**-20 + 2.0 * score_slack(big, D).unsqueeze(-1)) + want.abs() * 2.0**-11 + 2.0**-25
    assert bool(((got - want).abs() <= room).all()), float(((got - want).abs() / room).max())
