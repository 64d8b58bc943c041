"""fp16: what places hold that nothing sees, finite and as large as fp16 goes, does not move the power of two that the scores'
gradients are held by: outputs and gradients keep their bits."""
import pytest
import torch

import cdna4_sage
from test_gpu_train import _compare, _draw, _run
from train_util import Exact

pytestmark = pytest.mark.gpu

HF = torch.float16
LARGE = 6e4


def _same(a, b):
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for x, y in zip(a[2], b[2]):
        assert bool(torch.isfinite(y).all()) and torch.equal(x, y)


def _forms(B, H, Hkv, Sq, Skv):
    """(name, mask, causal): in each, some keys are seen by no query and some queries see nothing."""
    g = torch.Generator().manual_seed(3)
    yield "keys", (torch.arange(Skv) < torch.tensor([Skv - 70, 0, 65])[:B, None])[:, None, None], False
    yield "keys, causal", (torch.rand(B, 1, 1, Skv, generator=g) < 0.6), True
    heads = torch.zeros(1, H, Sq, Skv, dtype=torch.bool)
    heads[:, 1, ::2, 3:Skv:5] = True                  # only one of the heads that share its keys sees them
    heads[:, H - 1, 7, 11] = True
    yield "heads", heads, False
    late = torch.zeros(B, 1, Sq, Skv, dtype=torch.bool)
    late[:, :, :Sq // 2, Skv // 2:] = True            # with causal: pairs that only the mask would show
    late[:, :, :, :9] = True
    yield "late, causal", late, True
    yield "rows", torch.rand(Sq, Skv, generator=g) < 0.002, False


@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_masks(dev, D):
    B, H, Hkv, Sq, Skv = 3, 4, 2, 150, 260
    q, k, v, do = _draw(B, H, Hkv, Sq, Skv, D, HF, seed=41)
    for name, mask, causal in _forms(B, H, Hkv, Sq, Skv):
        vis = mask.expand(B, H, Sq, Skv)
        if causal:
            vis = vis & torch.ones(Sq, Skv, dtype=torch.bool).tril(Skv - Sq)
        keys = ~vis.unflatten(1, (Hkv, H // Hkv)).any(2).any(2)          # [B, Hkv, Skv] that nothing sees
        rows = ~vis.any(3)                                               # [B, H, Sq] that see nothing
        assert bool(keys.any()) and bool((~keys).any()), name
        kw = dict(attn_mask=mask.to(dev), is_causal=causal)
        want = _run(dev, q, k, v, do, **kw)
        _compare(Exact(q, k, v, causal=causal, seen=mask, dout=do), *want)
        for where in ("v", "do", "all"):
            ts = [t.clone() for t in (q, k, v, do)]
            for i, gone in enumerate((rows, keys, keys, rows)):
                if where == "all" or (where == "v" and i == 2) or (where == "do" and i == 3):
                    ts[i][gone] = LARGE
                    ts[i][..., 1] = torch.where(gone, -LARGE, ts[i][..., 1])
            _same(want, _run(dev, *ts, **kw))


def test_long_masks(dev):
    """More than 64 blocks of rows, the only one that sees a key among the last."""
    S, D = 64 * 66 + 3, 64
    mask = torch.zeros(S, S, dtype=torch.bool)
    mask[:, :40] = True
    mask[S - 2, 100] = True
    mask[64 * 64 + 1, 64 * 65] = True
    q, k, v, do = _draw(1, 1, 1, S, S, D, HF, seed=43)
    v[:, :, 100], v[:, :, 64 * 65] = 300.0, -200.0    # (they count)
    kw = dict(attn_mask=mask.to(dev))
    want = _run(dev, q, k, v, do, **kw)
    _compare(Exact(q, k, v, seen=mask, dout=do), *want)
    gone = ~mask.any(0)
    ts = [q, *(t.clone() for t in (k, v)), do]
    ts[1][:, :, gone], ts[2][:, :, gone] = LARGE, LARGE
    _same(want, _run(dev, *ts, **kw))


@pytest.mark.parametrize("D,causal", [(64, True), (96, False), (128, True), (256, False)])
def test_packed_gaps(dev, D, causal):
    """Rows that no sequence covers, keys of sequences without queries, queries of sequences without keys or before the first key."""
    H, Hkv = 4, 2
    lq, lk = [0, 70, 5, 130, 64], [90, 70, 0, 30, 65]
    first = 6
    cu = [torch.tensor([first] + [first + sum(n[:i + 1]) for i in range(len(n))], dtype=torch.int32) for n in (lq, lk)]
    TQ, TK = int(cu[0][-1]) + 9, int(cu[1][-1]) + 140
    g = torch.Generator().manual_seed(45)
    q, do = (torch.randn(TQ, H, D, generator=g).to(HF) for _ in range(2))
    k, v = (torch.randn(TK, Hkv, D, generator=g).to(HF) for _ in range(2))
    rows, keys = torch.ones(TQ, dtype=torch.bool), torch.ones(TK, dtype=torch.bool)
    for b, (n, m) in enumerate(zip(lq, lk)):
        if n and m:
            rows[int(cu[0][b]) + (max(0, n - m) if causal else 0):int(cu[0][b + 1])] = False
            keys[int(cu[1][b]):int(cu[1][b + 1])] = False

    def run(*ts):
        leaves = [t.to(dev).requires_grad_() for t in ts[:3]]
        out, lse = cdna4_sage.attention_train_varlen(*leaves, cu[0].to(dev), cu[1].to(dev), is_causal=causal, return_lse=True)
        inside = torch.zeros(TQ, dtype=torch.bool)
        inside[first:int(cu[0][-1])] = True
        return out, lse[:, inside.to(dev)], torch.autograd.grad(out, leaves, ts[3].to(dev))

    want = run(q, k, v, do)
    for where in ("v", "do", "all"):
        ts = [t.clone() for t in (q, k, v, do)]
        for i, gone in enumerate((rows, keys, keys, rows)):
            if where == "all" or (where == "v" and i == 2) or (where == "do" and i == 3):
                ts[i][gone] = LARGE
        _same(want, run(*ts))
    for b in (1, 4):
        r, c = slice(int(cu[0][b]), int(cu[0][b + 1])), slice(int(cu[1][b]), int(cu[1][b + 1]))
        one = [t[x].transpose(0, 1)[None] for t, x in ((q, r), (k, c), (v, c), (do, r))]
        e = Exact(*one[:3], causal=causal, dout=one[3])
        for got, exact, room in zip((want[0][r], want[2][0][r], want[2][1][c], want[2][2][c]), (e.out, e.dq, e.dk, e.dv),
                                    (e.room_out, e.room_dq + 1e-6, e.room_dk + 1e-6, e.room_dv)):
            assert bool(((got.transpose(0, 1)[None].double().cpu() - exact).abs() <= room).all())


def test_a_captured_step_whose_mask_changes(dev):
    """The keys that a mask shows are found anew at every replay."""
    B, H, Hkv, S, D = 2, 4, 2, 190, 64

    def draw(seed):
        q, k, v, do = _draw(B, H, Hkv, S, S, D, HF, seed=seed)
        shown = torch.arange(S) < torch.tensor([20 + 30 * (seed % 5), S - 40 * (seed % 3)])[:, None]
        v[~shown[:, None].expand(B, Hkv, S)] = LARGE
        return [t.to(dev) for t in (q, k, v, do, shown[:, None, None])]

    def step(q, k, v, do, mask):
        out = cdna4_sage.attention_train(q, k, v, attn_mask=mask, is_causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), do))

    held = [t.requires_grad_(i < 3) for i, t in enumerate(draw(50))]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*held)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for seed in (51, 52, 53, 54):
        new = draw(seed)
        want = step(*(t.clone().requires_grad_(i < 3) for i, t in enumerate(new)))
        clean = [t.clone() for t in new]
        clean[2][clean[2] == LARGE] = 0.0
        plain = step(*(t.requires_grad_(i < 3) for i, t in enumerate(clean)))
        noise = torch.randn(1 << 20, device=dev).sum()
        with torch.no_grad():
            for a, b in zip(held, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, plain))
        assert torch.isfinite(noise)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_the_largest_bf16_numbers_under_masks(dev, D):
    """Products with them pass float32: an infinity times a weight of 0 is none of what is seen."""
    B, H, Hkv, Sq, Skv = 3, 4, 2, 150, 260
    q, k, v, do = _draw(B, H, Hkv, Sq, Skv, D, torch.bfloat16, seed=47)
    for name, mask, causal in _forms(B, H, Hkv, Sq, Skv):
        vis = mask.expand(B, H, Sq, Skv)
        if causal:
            vis = vis & torch.ones(Sq, Skv, dtype=torch.bool).tril(Skv - Sq)
        keys, rows = ~vis.unflatten(1, (Hkv, H // Hkv)).any(2).any(2), ~vis.any(3)
        kw = dict(attn_mask=mask.to(dev), is_causal=causal)
        want = _run(dev, q, k, v, do, **kw)
        ts = [t.clone() for t in (q, k, v, do)]
        for t, gone in zip(ts, (rows, keys, keys, rows)):
            t[gone] = 3e38
            t[..., 2] = torch.where(gone, -3e38, t[..., 2])
        _same(want, _run(dev, *ts, **kw))


@pytest.mark.parametrize("D,dtype,large", [(64, HF, LARGE), (128, torch.bfloat16, 3e38), (256, HF, LARGE), (256, torch.bfloat16, 3e38)])
def test_queries_before_the_first_key(dev, D, dtype, large):
    """Causal, more queries than keys: without a mask, and with a bias inside."""
    q, k, v, do = _draw(2, 4, 2, 300, 170, D, dtype, seed=48)
    for bias in (None, torch.randn(16, 4, generator=torch.Generator().manual_seed(49)).to(dtype)):
        kw = dict(is_causal=True, table=bias)
        want = _run(dev, q, k, v, do, **kw)
        ts = [q.clone(), k, v, do.clone()]
        ts[0][:, :, :130], ts[3][:, :, :130] = large, -large
        _same(want, _run(dev, *ts, **kw))
