"""attention_train where the query heads of a kv head are shared out over workgroups, and at the farthest reach of a bias."""
import pytest
import torch

import cdna4_sage
from test_gpu_train import _compare, _draw, _run
from train_util import Exact, bucket_map, close

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D,dtype,layout,causal,masked", [
    (43, 12, 2, 100, 100, 128, BF, "HND", True, False),     # three workgroups of two heads: six would be more than fit at once
    (2, 6, 1, 150, 290, 96, HF, "NHD", True, False),
    (1, 8, 1, 64, 64, 256, BF, "HND", False, False),
    (30, 10, 2, 70, 90, 64, BF, "NHD", False, True),
    (1, 7, 1, 513, 300, 128, HF, "HND", False, True),
    (1, 16, 1, 5, 1, 64, HF, "NHD", False, False),
])
def test_heads_in_several_workgroups(dev, B, H, Hkv, Sq, Skv, D, dtype, layout, causal, masked):
    q, k, v, do = _draw(B, H, Hkv, Sq, Skv, D, dtype, seed=51)
    kw = {"is_causal": causal}
    if masked:      # by heads, one of which shows nothing
        kw["attn_mask"] = (torch.rand(1, H, Sq, Skv, generator=torch.Generator().manual_seed(52)) < 0.5)
        kw["attn_mask"][:, 1] = False
    e = Exact(q, k, v, causal=causal, seen=kw.get("attn_mask"), dout=do)
    kw = {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    out, lse, grads = _run(dev, q, k, v, do, layout, **kw)
    _compare(e, out, lse, grads)
    again = _run(dev, q, k, v, do, layout, **kw)
    assert all(torch.equal(a, b) for a, b in zip(grads, again[2]))


@pytest.mark.parametrize("D,dtype", [(64, HF), (96, BF), (128, BF), (256, BF), (256, HF)])
def test_the_farthest_reach_with_a_mask(dev, D, dtype):
    B, H, Hkv, S, buckets, far = 1, 2, 1, 900, 256, 790     # (the last bucket begins at 760)
    q, k, v, do = _draw(B, H, Hkv, S, S, D, dtype, seed=53)
    g = torch.Generator().manual_seed(54)
    table = torch.randn(buckets, H, generator=g).to(dtype)
    mask = torch.rand(1, 1, S, S, generator=g) < 0.7
    bucket = bucket_map(S, S, buckets, far, True)
    out, lse, grads = _run(dev, q, k, v, do, table=table, attn_mask=mask.to(dev), max_distance=far)
    e = Exact(q, k, v, seen=mask, bias=table.double()[bucket].permute(2, 0, 1), dout=do)
    _compare(e, out, lse, grads[:3])
    close(grads[3], *e.table(bucket, buckets, bucket % 128 == 127, dtype))
    with pytest.raises(cdna4_sage.Unsupported):
        _run(dev, q, k, v, do, table=table, max_distance=far + 1)


def test_captured_packed_steps_of_shared_heads(dev):
    """Forward and backward with a bias in one graph, replayed with other sequences and numbers."""
    T, H, Hkv, D = 700, 8, 2, 128

    def draw(seed):
        g = torch.Generator().manual_seed(seed)
        ts = [torch.randn(T, h, D, generator=g).to(BF).to(dev) for h in (H, Hkv, Hkv, H)]
        cu = torch.randint(0, T + 1, (5,), generator=g).sort().values.to(device=dev, dtype=torch.int32)
        return (*ts, torch.randn(32, H, generator=g).to(BF).to(dev), cu)

    def step(q, k, v, do, table, cu):
        out = cdna4_sage.attention_train_varlen(q, k, v, cu, cu, is_causal=True, bias_table=table, bidirectional=False)
        return (out, *torch.autograd.grad(out, (q, k, v, table), do))

    def leaves(ts):
        return [t.clone().requires_grad_(i in (0, 1, 2, 4)) for i, t in enumerate(ts[:5])] + [ts[5].clone()]

    held = leaves(draw(60))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*held)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for r in range(4):
        new = draw(61 + r)
        want = step(*leaves(new))
        noise = torch.randn(1 << 20, device=dev).sum()
        with torch.no_grad():
            for a, b in zip(held, new):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), r
        assert torch.isfinite(noise)


def test_offsets_that_pass_32_bits(dev):
    T, H, D = 40, 2, 64
    ts = [torch.randn(T, H, D, generator=torch.Generator().manual_seed(i)).to(BF).to(dev).requires_grad_() for i in range(3)]
    cu = torch.tensor([0, 15, 40], device=dev)
    want = cdna4_sage.attention_train_varlen(*ts, cu, cu.to(torch.int32))
    assert bool((want != 0).any())
    for bad in (torch.tensor([0, 15, 40 + (1 << 32)]), torch.tensor([0, 15 - (1 << 32), 40])):
        out = cdna4_sage.attention_train_varlen(*ts, bad.to(dev), cu)
        grads = torch.autograd.grad(out, ts, torch.ones_like(out))
        assert all(bool((t == 0).all()) for t in (out, *grads))
    for other in (torch.float32, torch.int16, torch.bool):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.attention_train_varlen(*ts, cu.to(other), cu)


def test_the_ops_check_what_callers_bring(dev):
    op = torch.ops.cdna4_sage
    q, k, v, do = (torch.randn(1, 2, 70, 64, generator=torch.Generator().manual_seed(i)).to(BF).to(dev) for i in range(4))
    how = ("HND", 0.0, False, True, 128)
    out, lse, state = op.attention_train(q, k, v, None, None, None, None, *how, True)
    good = [do, q, k, v, out, lse, state, None, None, None, *how, []]
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(cdna4_sage.attention_train(*leaves), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(op.attention_train_backward(*good)[:3], want))
    for place, bad in ((0, do[:, :1]), (0, do.float()), (0, do.cpu()), (4, out[:, :, :69]), (5, lse[:, :, :69]), (5, lse.double()),
                       (5, lse.cpu()), (6, state[:16]), (6, state.cpu()), (15, [1]), (15, [1, 1, 1])):
        with pytest.raises(cdna4_sage.Unsupported):
            op.attention_train_backward(*good[:place], bad, *good[place + 1:])
    rows = [t[0].transpose(0, 1) for t in (q, k, v)]
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=dev)
    for a, b in ((cu.long(), cu), (cu, None), (None, cu), (cu.cpu(), cu), (cu, cu[:2]), (cu[:1], cu[:1])):
        with pytest.raises(cdna4_sage.Unsupported):
            op.attention_train(*(rows if a is not None else (q, k, v)), None, None, a, b, *how, False)
