"""cache_attention's sharing of work: every XCD its part for any number of kv heads, and tables wider than the sequences are
long.  Times are compared within one run, in turn, with wide margins."""
import pytest
import torch

import cdna4_sage
from cache_util import attention, attention_slack, random_cache
from test_gpu_cache import _compare, _table, _tree

pytestmark = pytest.mark.gpu


def _times(calls, n=20):
    """GPU time of n calls of each, back to back: the medians of 7 rounds in turn, in us a call."""
    for call in calls:
        for _ in range(3):
            call()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    out = [[] for _ in calls]
    for _ in range(7):
        for call, times in zip(calls, out):
            torch.cuda.synchronize()
            start.record()
            for _ in range(n):
                call()
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end) * 1e3 / n)
    return [sorted(t)[3] for t in out]


def _prompt(dev, T, Hkv, columns=0, B=1, D=128, H=None):
    page = 16
    need = -(-T // page)
    cache = cdna4_sage.new_cache(B * need, page, Hkv, D, device=dev)
    k = torch.randn(B * T, Hkv, D, device=dev).to(torch.bfloat16)
    table = torch.full((B, max(need, columns)), -1, dtype=torch.int32)
    table[:, :need] = torch.arange(B * need).view(B, need)
    table, lengths = table.to(dev), torch.full((B,), T, dtype=torch.int32, device=dev)
    cdna4_sage.cache_write(cache, k, k, cdna4_sage.cache_slots(table, lengths, T, page).view(-1))
    q = torch.randn(B, 4 * Hkv if H is None else H, T, D, device=dev).to(torch.bfloat16)
    return lambda: cdna4_sage.cache_attention(q, cache, table, lengths)


def test_few_heads_use_the_whole_card(dev):
    """An eighth (a quarter) of the work of eight kv heads takes far less than their time."""
    one, two, eight = _times([_prompt(dev, 2048, h) for h in (1, 2, 8)])
    assert one < 0.7 * eight and two < 0.7 * eight, (one, two, eight)


@pytest.mark.parametrize("T, H, Hkv, D, columns", [
    (19, 6, 3, 64, 0), (70, 5, 5, 128, 0), (33, 11, 11, 96, 0), (150, 3, 3, 256, 0), (64, 9, 9, 128, 0), (40, 12, 12, 64, 300),
    (55, 10, 10, 128, 700), (21, 7, 7, 256, 400), (9, 13, 13, 96, 64), (130, 1, 1, 128, 40)])
def test_every_number_of_ranges(dev, T, H, Hkv, D, columns):
    """Numbers of kv heads, ranges and row blocks that eight does not divide: each item is done once."""
    g = torch.Generator().manual_seed(T)
    lengths = torch.tensor([T, T + 170, 0], dtype=torch.int32)
    page = 16
    pages = sum(-(-int(x) // page) for x in lengths) + 1
    cache = random_cache(g, pages, page, Hkv, D, torch.int8)
    q = torch.randn(3, H, T, D, generator=g).to(torch.bfloat16)
    _compare(dev, q, cache, _table(g, lengths, page, pages, columns=columns or None), lengths, tree=_tree(g, 3, T) if T % 2 else None)


def test_a_wide_table_costs_little(dev):
    """Prompts with a table as wide as a captured step keeps it, against one of their own width."""
    for T in (1024, 2048):
        narrow, wide = _times([_prompt(dev, T, 8), _prompt(dev, T, 8, 8192)])
        assert wide < 1.7 * narrow, (T, narrow, wide)


def test_workspaces_stay_small(dev):
    from cdna4_sage import _capi

    for B, H, Hkv, T, D in ((1, 32, 8, 2048, 128), (1, 64, 8, 8192, 128), (16, 32, 8, 8192, 128), (1, 24, 24, 4096, 96),
                            (2, 16, 4, 8192, 64), (1, 12, 12, 4096, 256), (1, 32, 8, 512, 128), (64, 32, 8, 1, 128)):
        for columns in (64, 512, 8192, 65536):
            assert _capi.cache_attn_workspace(B, H, Hkv, T, D, 16, columns) <= 2**28, (B, H, T, columns)


@pytest.mark.parametrize("B, T, H, Hkv, D, longest, columns", [
    (2, 300, 8, 8, 128, 2600, (0, 2000)),      # few sequences' walks: several ranges, or one, by the lengths
    (1, 350, 6, 6, 96, 350, (0, 4096)),
    (1, 700, 6, 3, 64, 1900, (0, 2048)),
    (3, 200, 6, 6, 256, 900, (0, 1024)),
    (66, 65, 12, 12, 256, 130, (600,)),        # more sequences than lanes
])
def test_ranges_follow_the_lengths(dev, B, T, H, Hkv, D, longest, columns):
    g = torch.Generator().manual_seed(T + D)
    lengths = torch.randint(T // 2, longest + 1, (B,), generator=g).to(torch.int32)
    lengths[0] = longest
    page = 16
    pages = sum(-(-int(x) // page) for x in lengths) + 1
    cache = random_cache(g, pages, page, Hkv, D, torch.int8)
    q = torch.randn(B, H, T, D, generator=g).to(torch.bfloat16)
    for n in columns:
        _compare(dev, q, cache, _table(torch.Generator().manual_seed(1), lengths, page, pages, columns=n or None), lengths)


def test_replays_whose_lengths_change_the_ranges(dev):
    """A captured chunk with a wide table, replayed with lengths of one range and of several: every replay as the eager call and
    as float64 attention."""
    g = torch.Generator().manual_seed(3)
    B, T, H, Hkv, D, page, columns = 2, 300, 8, 8, 128, 64, 300
    pages = 120
    cache = random_cache(g, pages, page, Hkv, D, torch.int8)
    q = torch.randn(B, H, T, D, generator=g).to(torch.bfloat16)
    need = torch.randperm(pages, generator=g).to(torch.int32).view(B, 60)
    table = torch.cat([need, torch.full((B, columns - 60), -1, dtype=torch.int32)], 1)
    on = [cdna4_sage.KVCache(*(t.to(dev) for t in cache)), q.to(dev), table.to(dev),
          torch.tensor([T, T], dtype=torch.int32, device=dev)]
    call = lambda: cdna4_sage.cache_attention(on[1], on[0], on[2], on[3], return_lse=True)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for lengths in ([T, T], [3800, 300], [0, 0], [3840, 3840], [1, 900], [T, T]):
        on[3].copy_(torch.tensor(lengths, dtype=torch.int32))
        want = call()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), lengths
    on[3].copy_(torch.tensor([3800, 300], dtype=torch.int32))
    few = attention(q[:, :2].double(), [t[:, :2] for t in cache], table, torch.tensor([3800, 300]))
    off = (call()[0][:, :2].double().cpu() - few[0]).abs()
    assert bool((off <= attention_slack(few[2], few[3], few[0], D, q.dtype)).all())
