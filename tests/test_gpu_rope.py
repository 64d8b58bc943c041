"""cdna4_sage.rope against the rotation in float64: both pair layouts, parts of the head, far positions, strides, single
tokens and many heads; gradients against the formula and against differences; streams, graphs, torch.compile."""
import pytest
import torch

import cdna4_sage
from cache_util import rotate, rotate_slack

pytestmark = pytest.mark.gpu


def _inputs(B, S, H, Hk, D, dtype, layout, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for h in (H, Hk):
        x = torch.randn(B, S, h, D, generator=g).to(dtype)
        out.append(x)
    return out


def _check(got, x, positions, freqs, interleaved, factor, back=False):
    want, m = rotate(x.double(), positions, freqs, interleaved, factor, back)
    off = (got.double().cpu() - want).abs()
    room = rotate_slack(want, m, factor, x.dtype)
    assert bool((off <= room).all()), float((off / room.clamp(min=1e-30)).max())


CASES = [
    # B, S, H, Hk, D, rot, dtype, layout, interleaved
    (1, 1, 8, 2, 128, 128, torch.bfloat16, "NHD", False),
    (3, 37, 6, 2, 64, 64, torch.float16, "HND", False),
    (2, 19, 5, 1, 96, 24, torch.bfloat16, "NHD", False),
    (2, 19, 5, 1, 96, 24, torch.float16, "HND", True),
    (1, 130, 12, 12, 256, 64, torch.bfloat16, "HND", False),
    (2, 33, 4, 3, 128, 8, torch.bfloat16, "NHD", True),
    (1, 77, 24, 24, 128, 128, torch.float16, "NHD", True),
    (5, 1, 32, 8, 64, 32, torch.bfloat16, "HND", True),
    (2, 700, 32, 8, 128, 128, torch.bfloat16, "NHD", False),   # several heads per thread
    (2, 1500, 20, 5, 128, 64, torch.float16, "HND", True),
]


@pytest.mark.parametrize("B,S,H,Hk,D,rot,dtype,layout,interleaved", CASES)
def test_rope_matches_float64(dev, B, S, H, Hk, D, rot, dtype, layout, interleaved):
    q, k = _inputs(B, S, H, Hk, D, dtype, layout)
    g = torch.Generator().manual_seed(9)
    positions = torch.randint(0, 200000, (B, S), generator=g)
    freqs, factor = cdna4_sage.rope_frequencies(rot, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096})
    put = lambda t: (t.transpose(1, 2).contiguous() if layout == "HND" else t).to(dev)  # noqa: E731
    oq, ok = cdna4_sage.rope(put(q), put(k), positions.to(dev), freqs.to(dev), layout, interleaved, factor)
    back = lambda t: t.transpose(1, 2) if layout == "HND" else t  # noqa: E731
    assert oq.dtype == dtype and oq.shape == put(q).shape
    _check(back(oq), q, positions, freqs, interleaved, factor)
    _check(back(ok), k, positions, freqs, interleaved, factor)
    # q alone, int32 positions
    one = cdna4_sage.rope(put(q), None, positions.to(dev, torch.int32), freqs.to(dev), layout, interleaved, factor)
    assert torch.equal(one, oq)


def test_positions_shared_default_negative_and_far(dev):
    B, S, H, D = 2, 11, 3, 64
    q, _ = _inputs(B, S, H, 1, D, torch.float16, "NHD")
    freqs, _ = cdna4_sage.rope_frequencies(D)
    qd, fd = q.to(dev), freqs.to(dev)
    _check(cdna4_sage.rope(qd, None, None, fd, "NHD"), q, torch.arange(S).expand(B, S), freqs, False, 1.0)
    for p in (torch.arange(S) - 5, torch.arange(S) + 2**33, torch.full((S,), 2**31 - 1)):
        got = cdna4_sage.rope(qd, None, p.to(dev), fd, "NHD")
        # the 64-bit product of the position and the frequency itself is off by 2^-53 of the angle
        want, m = rotate(q.double(), p.expand(B, S), freqs, False)
        room = rotate_slack(want, m, 1.0, q.dtype) + m * float(p.abs().max()) * 2.0**-51
        assert bool(((got.double().cpu() - want).abs() <= room).all())
    p = torch.arange(S * B).reshape(S, B).to(dev).t()          # [B, S] with swapped strides
    _check(cdna4_sage.rope(qd, None, p, fd, "NHD"), q, p.cpu(), freqs, False, 1.0)


def test_strided_inputs_keep_their_order_and_neighbours(dev):
    B, S, H, D = 2, 9, 4, 128
    fused = torch.randn(B, S, 3 * H * D, device=dev).to(torch.bfloat16)
    q = fused[..., :H * D].unflatten(-1, (H, D))               # a slice of a fused projection
    k = fused[..., H * D:2 * H * D].unflatten(-1, (H, D))
    before = fused.clone()
    freqs, _ = cdna4_sage.rope_frequencies(D)
    oq, ok = cdna4_sage.rope(q.transpose(1, 2), k.transpose(1, 2), None, freqs.to(dev), "HND")
    pos = torch.arange(S).expand(B, S)
    _check(oq.transpose(1, 2), q.cpu(), pos, freqs, False, 1.0)
    _check(ok.transpose(1, 2), k.cpu(), pos, freqs, False, 1.0)
    assert torch.equal(fused, before)
    odd = torch.randn(B * S * H * D + 1, device=dev).to(torch.bfloat16)[1:].view(B, S, H, D)   # misaligned base
    _check(cdna4_sage.rope(odd, None, None, freqs.to(dev), "NHD"), odd.cpu(), pos, freqs, False, 1.0)
    wide = torch.randn(B, S, H, D, device=dev).to(torch.bfloat16).expand(B, S, H, D)[:, :, :1].expand(B, S, H, D)
    _check(cdna4_sage.rope(wide, None, None, freqs.to(dev), "NHD"), wide.cpu(), pos, freqs, False, 1.0)


def test_empty_and_unturned_values(dev):
    freqs, _ = cdna4_sage.rope_frequencies(64)
    q = torch.empty(0, 5, 4, 64, dtype=torch.bfloat16, device=dev)
    assert cdna4_sage.rope(q, None, None, freqs.to(dev), "NHD").shape == q.shape
    q = torch.empty(2, 0, 4, 64, dtype=torch.bfloat16, device=dev)
    assert cdna4_sage.rope(q, q, None, freqs.to(dev), "NHD")[1].shape == q.shape
    q = torch.randn(1, 3, 2, 256, device=dev).to(torch.float16)
    q[0, 1, 0, 200], q[0, 2, 1, 3] = float("inf"), float("nan")
    out = cdna4_sage.rope(q, None, None, freqs.to(dev), "NHD")
    assert torch.equal(out[..., 64:], q[..., 64:])             # copied bit for bit, infinity among them
    assert bool(torch.isnan(out[0, 2, 1, [3, 35]]).all()) and bool(torch.isfinite(out[0, 0]).all())


@pytest.mark.parametrize("interleaved,rot", [(False, 64), (True, 32), (False, 24)])
def test_gradients_match_formula_and_differences(dev, interleaved, rot):
    B, S, H, Hk, D = 2, 5, 4, 2, 64
    q, k = _inputs(B, S, H, Hk, D, torch.float16, "NHD", seed=3)
    dq, dk = _inputs(B, S, H, Hk, D, torch.float16, "NHD", seed=4)
    freqs, _ = cdna4_sage.rope_frequencies(rot)
    factor = 1.25
    pos = torch.arange(S).expand(B, S) + 1000
    a, b = (t.to(dev).requires_grad_(True) for t in (q, k))
    oq, ok = cdna4_sage.rope(a, b, pos.to(dev), freqs.to(dev), "NHD", interleaved, factor)
    ga, gb = torch.autograd.grad((oq, ok), (a, b), (dq.to(dev), dk.to(dev)), create_graph=True)
    _check(ga, dq, pos, freqs, interleaved, factor, back=True)
    _check(gb, dk, pos, freqs, interleaved, factor, back=True)
    # differences: the map is linear, so <g, f(x + e) - f(x)> = <grad, e> in exact arithmetic
    e = torch.randn(q.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    f = lambda x: rotate(x, pos, freqs, interleaved, factor)[0]  # noqa: E731
    change = float(((f(q.double() + e) - f(q.double())) * dq.double()).sum())
    slack = float((e.abs() * (ga.detach().double().cpu().abs() * 2.0**-11 + 2.0**-17)).sum())
    assert abs(change - float((ga.detach().double().cpu() * e).sum())) <= slack
    # only one of the two, a broadcast gradient, and the gradient of a gradient (the rotation itself)
    oq, ok = cdna4_sage.rope(a, b.detach(), pos.to(dev), freqs.to(dev), "NHD", interleaved, factor)
    (g1,) = torch.autograd.grad(oq, a, dq.to(dev))
    assert torch.equal(g1, ga.detach())
    oq = cdna4_sage.rope(a, None, pos.to(dev), freqs.to(dev), "NHD", interleaved, factor)
    (g2,) = torch.autograd.grad(oq.sum(), a)
    _check(g2, torch.ones_like(q), pos, freqs, interleaved, factor, back=True)
    u = torch.ones(B, S, H, D, dtype=torch.float16, device=dev, requires_grad=True)
    (g3,) = torch.autograd.grad(cdna4_sage.rope(a, None, pos.to(dev), freqs.to(dev), "NHD", interleaved, factor), a, u,
                                create_graph=True)
    (g4,) = torch.autograd.grad(g3, u, dq.to(dev))
    _check(g4, dq, pos, freqs, interleaved, factor)


@pytest.mark.parametrize("D, rot, interleaved", [(128, 128, False), (64, 24, False), (96, 40, True)])
def test_many_tokens_as_in_small_calls(dev, D, rot, interleaved):
    """Calls that turn several heads per thread: bit for bit what small ones give, for heads that are no multiple of them."""
    H, Hk, S = 11, 3, 5303
    q, k = (t.to(dev) for t in _inputs(1, S, H, Hk, D, torch.bfloat16, "NHD"))
    freqs = cdna4_sage.rope_frequencies(rot)[0].to(dev)
    pos = torch.arange(S, device=dev) * 37 - 1000
    got = cdna4_sage.rope(q, k, pos, freqs, "NHD", interleaved)
    for i in range(0, S, 700):
        want = cdna4_sage.rope(q[:, i:i + 700], k[:, i:i + 700], pos[i:i + 700], freqs, "NHD", interleaved)
        for a, b in zip(got, want):
            assert torch.equal(a[:, i:i + 700], b)


def test_refusals(dev):
    q, k = (t.to(dev) for t in _inputs(2, 8, 4, 2, 64, torch.bfloat16, "NHD"))
    freqs = cdna4_sage.rope_frequencies(64)[0].to(dev)
    pos = torch.arange(8, device=dev)
    ok = dict(q=q, k=k, positions=pos, freqs=freqs, tensor_layout="NHD")
    cdna4_sage.rope(**ok)
    for kw in (dict(q=q.float()), dict(k=k.half()), dict(q=q[0]), dict(k=k[0]), dict(k=k[:1]), dict(k=k[:, :7]), dict(k=k.cpu()),
               dict(q=q[..., :32], k=None), dict(freqs=None), dict(freqs=freqs.float()), dict(freqs=freqs[:3]),
               dict(freqs=freqs.cpu()), dict(freqs=torch.cat([freqs, freqs])), dict(positions=pos.float()),
               dict(positions=pos[:7]), dict(positions=pos.cpu()), dict(positions=pos.expand(3, 8)), dict(tensor_layout="x")):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.rope(**{**ok, **kw})


def test_training_step_in_a_graph(dev):
    q, k = (t.to(dev).requires_grad_(True) for t in _inputs(2, 40, 6, 2, 64, torch.float16, "HND"))
    freqs = cdna4_sage.rope_frequencies(32)[0].to(dev)
    pos = torch.arange(40, device=dev)
    dq, dk = (torch.randn_like(t) for t in (q, k))

    def step():
        out = cdna4_sage.rope(q, k, pos, freqs, "NHD")
        return torch.autograd.grad(out, (q, k), (dq, dk.mean(2, keepdim=True).expand_as(k)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        pos.add_(11), dq.mul_(-0.5)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


def test_stream_and_graph(dev):
    B, S, H, Hk, D = 2, 64, 8, 2, 128
    q, k = (t.to(dev) for t in _inputs(B, S, H, Hk, D, torch.bfloat16, "NHD"))
    freqs = cdna4_sage.rope_frequencies(D)[0].to(dev)
    pos = torch.arange(S, device=dev).expand(B, S).contiguous()
    eager = cdna4_sage.rope(q, k, pos, freqs, "NHD")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cdna4_sage.rope(q, k, pos, freqs, "NHD")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], eager[0]) and torch.equal(other[1], eager[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cdna4_sage.rope(q, k, pos, freqs, "NHD")
    for i in range(3):
        pos.add_(7)
        want = cdna4_sage.rope(q, k, pos, freqs, "NHD")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i


def test_traced(dev):
    q, k = (t.to(dev) for t in _inputs(1, 16, 4, 2, 64, torch.bfloat16, "NHD"))
    freqs = cdna4_sage.rope_frequencies(64)[0].to(dev)
    want = cdna4_sage.rope(q, k, None, freqs, "NHD")
    fn = torch.compile(lambda a, b: cdna4_sage.rope(a, b, None, freqs, "NHD"), backend="aot_eager", fullgraph=True)
    got = fn(q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a = q.clone().requires_grad_(True)
    one = torch.compile(lambda x: cdna4_sage.rope(x, None, None, freqs, "NHD"), backend="aot_eager", fullgraph=True)(a)
    (ga,) = torch.autograd.grad(one, a, q)
    b = q.clone().requires_grad_(True)
    (gb,) = torch.autograd.grad(cdna4_sage.rope(b, None, None, freqs, "NHD"), b, q)
    assert torch.equal(ga, gb)
