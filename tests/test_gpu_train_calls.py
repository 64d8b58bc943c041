"""How attention_train and relative_bias are called: strides, broadcast inputs, leaves without gradients, streams, captured
graphs, tracers, empty tensors; and the bias alone against whole numbers and float64."""
import math

import pytest
import torch

import cdna4_sage
from train_util import F32, Exact, bucket_map, close, half_step

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, seed, dtype=BF):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _grads(out, leaves, do):
    return torch.autograd.grad(out, leaves, do, retain_graph=True)


# ---- tensors as callers have them -----------------------------------------------------------------------------------------

def test_slices_of_one_projection_and_odd_bases(dev):
    B, S, H, D = 2, 130, 4, 64
    x = _rand((B, S, 3, H, D), 1).to(dev).requires_grad_()
    q, k, v = x.unbind(2)
    out = cdna4_sage.attention_train(q, k, v, "NHD", is_causal=True)
    do = _rand((B, S, H, D), 2).to(dev)
    dx, = _grads(out, [x], do)
    leaves = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    want = cdna4_sage.attention_train(*leaves, "NHD", is_causal=True)
    assert torch.equal(out, want)
    for a, b in zip(dx.unbind(2), _grads(want, leaves, do)):
        assert torch.equal(a, b)
    # off 16-byte boundaries, channels not innermost, a gradient of one number everywhere
    odd = torch.empty(B * S * H * D + 1, dtype=BF, device=dev)[1:].view(B, S, H, D).copy_(q.detach()).requires_grad_()
    turned = k.detach().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    out = cdna4_sage.attention_train(odd, turned, v.detach(), "NHD", is_causal=True)
    assert torch.equal(out, want)
    g = out.sum()
    a = torch.autograd.grad(g, [odd, turned])
    b = _grads(want, leaves[:2], torch.ones_like(want))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_broadcast_keys_and_rows_far_apart(dev):
    B, H, S, D = 3, 2, 100, 128
    q, do = (_rand((B, H, S, D), s).to(dev) for s in (3, 4))
    k, v = (_rand((1, H, S, D), s).to(dev).requires_grad_() for s in (5, 6))
    out = cdna4_sage.attention_train(q, k.expand(B, H, S, D), v.expand(B, H, S, D))
    dk, dv = _grads(out, [k, v], do)
    e = Exact(q.cpu(), k.detach().cpu().expand(B, H, S, D), v.detach().cpu().expand(B, H, S, D), dout=do.cpu())
    close(dk, e.dk.sum(0, keepdim=True), e.room_dk.sum(0, keepdim=True) + 4 * half_step(BF) * e.dk.abs().sum(0, keepdim=True))
    close(dv, e.dv.sum(0, keepdim=True), e.room_dv.sum(0, keepdim=True) + 4 * half_step(BF) * e.dv.abs().sum(0, keepdim=True))
    # rows so far apart that a tile's offsets pass 32 bits
    far = torch.empty(80 * (1 << 24) + 64, dtype=BF, device=dev).as_strided((1, 1, 80, 64), (0, 0, 1 << 24, 1))
    near = _rand((1, 1, 80, 64), 7).to(dev)
    far.copy_(near)
    for args in ((far, near, near), (near, far, far)):
        leaves = [t.requires_grad_() if t is near else t for t in args]
        got = cdna4_sage.attention_train(*leaves, is_causal=True)
        assert torch.equal(got, cdna4_sage.attention_train(near, near, near, is_causal=True))
    dq, = torch.autograd.grad(cdna4_sage.attention_train(near, far, far, is_causal=True), [near], near.detach())
    other = near.detach().clone().requires_grad_()
    assert torch.equal(dq, torch.autograd.grad(cdna4_sage.attention_train(other, near.detach(), near.detach(), is_causal=True), [other],
                                               near.detach())[0])


def test_only_the_gradients_that_are_asked_for(dev):
    q, k, v, do = (_rand((1, 2, 90, 64), s).to(dev) for s in range(8, 12))
    table = _rand((16, 2), 13).to(dev)
    full = [t.clone().requires_grad_() for t in (q, k, v, table)]
    want = _grads(cdna4_sage.attention_train(*full[:3], bias_table=full[3]), full, do)
    for i in range(4):
        ts = [q, k, v, table]
        ts[i] = ts[i].clone().requires_grad_()
        out = cdna4_sage.attention_train(*ts[:3], bias_table=ts[3])
        assert torch.equal(_grads(out, [ts[i]], do)[0], want[i])
    with torch.no_grad():
        assert not cdna4_sage.attention_train(*full[:3]).requires_grad
    # a logsumexp has no gradient, a second derivative neither
    out, lse = cdna4_sage.attention_train(*full[:3], return_lse=True)
    assert not lse.requires_grad
    d, = torch.autograd.grad(out.sum(), full[:1], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_no_tokens(dev):
    for shape_q, shape_k in (((0, 2, 5, 64), (0, 2, 5, 64)), ((1, 2, 0, 64), (1, 2, 5, 64)), ((1, 2, 5, 64), (1, 2, 0, 64)),
                             ((1, 0, 5, 64), (1, 2, 5, 64))):
        q = torch.zeros(shape_q, dtype=BF, device=dev, requires_grad=True)
        k, v = (torch.ones(shape_k, dtype=BF, device=dev, requires_grad=True) for _ in range(2))
        out, lse = cdna4_sage.attention_train(q, k, v, return_lse=True)
        assert out.shape == q.shape and bool((out == 0).all()) and bool((lse == -math.inf).all())
        for t, d in zip((q, k, v), _grads(out, [q, k, v], torch.ones_like(out))):
            assert d.shape == t.shape and bool((d == 0).all())
    table = torch.zeros(8, 3, device=dev, requires_grad=True)
    assert cdna4_sage.relative_bias(table, 0, 9).shape == (3, 0, 9)
    b = cdna4_sage.relative_bias(table, 4, 0)
    assert bool((torch.autograd.grad(b.sum(), table)[0] == 0).all())


def test_other_threads_streams_and_a_changed_input(dev):
    q, k, v, do = (_rand((2, 4, 300, 128), s).to(dev) for s in range(20, 24))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = cdna4_sage.attention_train(*leaves, is_causal=True)
    want = (out, *_grads(out, leaves, do))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                own = [t.clone().requires_grad_() for t in (q, k, v)]
                o = cdna4_sage.attention_train(*own, is_causal=True)
                got[i].append((o, *_grads(o, own, do)))
    torch.cuda.synchronize()
    for each in got:
        for r in each:
            assert all(torch.equal(a, b) for a, b in zip(r, want))
    # an input that was written to between the passes is noticed
    own = [t.clone().requires_grad_() for t in (q, k, v)]
    x = own[0] * 1.0
    o = cdna4_sage.attention_train(x, *own[1:])
    with torch.no_grad():
        x.zero_()
    with pytest.raises(RuntimeError):
        o.sum().backward()


def test_captured_steps(dev):
    """Forward and backward in one graph, dense with a mask and a bias and packed, replayed with new numbers; eager work between."""
    B, H, S, D = 2, 2, 200, 64
    q, k, v, do = (_rand((B, H, S, D), s).to(dev) for s in range(30, 34))
    table = _rand((32, H), 35).to(dev)
    mask = (torch.rand(B, 1, 1, S, generator=torch.Generator().manual_seed(36)) < 0.8).to(dev)
    cu = torch.tensor([0, 50, 50, 170, 200], dtype=torch.int32, device=dev)

    def dense(q, k, v, table, mask, cu, do):
        out = cdna4_sage.attention_train(q, k, v, attn_mask=mask, bias_table=table)
        return (out, *torch.autograd.grad(out, (q, k, v, table), do))

    def packed(q, k, v, table, mask, cu, do):
        rows = [t[0].transpose(0, 1) for t in (q, k, v)]
        out = cdna4_sage.attention_train_varlen(*rows, cu, cu, is_causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), do[0].transpose(0, 1)))

    for fn in (dense, packed):
        def leaves(seed):
            ts = [t.clone() for t in (q, k, v, table)]
            if seed:
                ts = [_rand(t.shape, seed + i).to(dev) for i, t in enumerate(ts)]
            return ts

        held = [t.requires_grad_() for t in leaves(0)]
        args = (*held, mask.clone(), cu.clone(), do.clone())
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fn(*args)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = fn(*args)
        for r in range(4):
            new = leaves(40 + 10 * r)
            m = (torch.rand(B, 1, 1, S, generator=torch.Generator().manual_seed(r)) < 0.6).to(dev)
            c = torch.tensor([0, 10 + r, 90, 90 + 5 * r, 200], dtype=torch.int32, device=dev)
            want = fn(*(t.clone().requires_grad_() for t in new), m, c, do)
            noise = torch.randn(1 << 20, device=dev).sum()
            with torch.no_grad():
                for a, b in zip(args, (*new, m, c)):
                    a.copy_(b)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), r
            assert torch.isfinite(noise)


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_traced(dev, layout):
    B, H, S, D = 2, 4, 70, 96
    shape = (B, H, S, D) if layout == "HND" else (B, S, H, D)
    q, k, v, do = (_rand(shape, s).to(dev) for s in range(50, 54))
    table = _rand((16, H), 54).to(dev)
    mask = (torch.rand(B, 1, 1, S, generator=torch.Generator().manual_seed(55)) < 0.7).to(dev)
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=dev)

    def fn(q, k, v, table):
        out, lse = cdna4_sage.attention_train(q, k, v, layout, attn_mask=mask, bias_table=table, return_lse=True)
        rows = [(t[0] if layout == "NHD" else t[0].transpose(0, 1)) for t in (q, k, v)]
        more = cdna4_sage.attention_train_varlen(*rows, cu, cu, is_causal=True)
        bias = cdna4_sage.relative_bias(table, 5, 9, dtype=torch.float32)
        return (out * do).sum() + more.float().square().sum() + bias.square().sum(), out, lse

    def run(f):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        loss, out, lse = f(*leaves)
        return (out, lse, *torch.autograd.grad(loss, leaves))

    want = run(fn)
    got = run(torch.compile(fn, backend="aot_eager", fullgraph=True))
    for a, b in zip(want, got):
        assert torch.equal(a, b) and a.stride() == b.stride()
    ops = torch.ops.cdna4_sage
    t = [x.clone().requires_grad_() for x in (q, k, v, table)]
    # (the full comparison of outputs would also compare what lies between the parts of the state, which nothing writes)
    torch.library.opcheck(ops.attention_train.default, (*t[:3], mask, t[3], None, None, layout, 0.0, False, True, 128, True),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    torch.library.opcheck(ops.relative_bias.default, (t[3], 5, 9, True, 128, torch.float32, 4, None))


def test_forward_mode_raises(dev):
    q = _rand((1, 1, 8, 64), 60).to(dev)
    table = _rand((8, 1), 61).to(dev)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            cdna4_sage.attention_train(dual, q, q)
        with pytest.raises(NotImplementedError):
            cdna4_sage.relative_bias(torch.autograd.forward_ad.make_dual(table, torch.ones_like(table)), 3, 3)


def test_refusals_on_the_device(dev):
    q = torch.zeros(1, 2, 8, 64, dtype=BF, device=dev)
    U = cdna4_sage.Unsupported
    for call in (lambda: cdna4_sage.attention_train(q, q, q, attn_mask=torch.zeros(8, 8, dtype=BF, device=dev)),
                 lambda: cdna4_sage.attention_train(q, q, q, attn_mask=torch.zeros(8, 8, dtype=torch.bool)),
                 lambda: cdna4_sage.attention_train(q, q, q, attn_mask=torch.zeros(3, 8, dtype=torch.bool, device=dev)),
                 lambda: cdna4_sage.attention_train(q, q, q, bias_table=torch.zeros(16, 3, dtype=BF, device=dev)),
                 lambda: cdna4_sage.attention_train(q, q, q, bias_table=torch.zeros(15, 2, dtype=BF, device=dev)),
                 lambda: cdna4_sage.attention_train(q, q, q, bias_table=torch.zeros(16, 2, dtype=BF, device=dev), max_distance=4),
                 lambda: cdna4_sage.attention_train(q, q, q, bias_table=torch.zeros(16, 2, dtype=BF, device=dev), max_distance=5000),
                 lambda: cdna4_sage.attention_train(q, q, q, sm_scale=math.inf),
                 lambda: cdna4_sage.attention_train(q, q, q[:, :, :4]),
                 lambda: cdna4_sage.attention_train(q, q, q.half()),
                 lambda: cdna4_sage.attention_train(q, torch.zeros(1, 3, 8, 64, dtype=BF, device=dev),
                                                    torch.zeros(1, 3, 8, 64, dtype=BF, device=dev)),
                 lambda: cdna4_sage.attention_train(q[..., :32], q[..., :32], q[..., :32]),
                 lambda: cdna4_sage.relative_bias(torch.zeros(16, 2, device=dev), 4, 4, q_offset=torch.zeros(1, device=dev)),
                 lambda: cdna4_sage.relative_bias(torch.zeros(16, 2, device=dev), 4, 4, dtype=torch.float64),
                 lambda: cdna4_sage.relative_bias(torch.zeros(16, 2, device=dev), -1, 4)):
        with pytest.raises(U):
            call()


# ---- the bias alone -------------------------------------------------------------------------------------------------------

BIAS = [
    # H, Sq, Skv, buckets, reach, two-sided, dtype, table type, offset
    (1, 1, 1, 4, 2, True, FF, FF, None),
    (3, 1, 300, 32, 128, False, BF, BF, None),
    (2, 65, 130, 32, 128, True, HF, FF, None),
    (2, 200, 17, 16, 9, True, BF, FF, None),
    (2, 130, 67, 2, 5, False, FF, HF, 1000),
    (1, 70, 2500, 64, 800, True, HF, HF, -300),
    (2, 33, 300, 256, 5000, True, FF, FF, 2 ** 40),
    (2, 129, 2048, 255, 129, False, BF, BF, -2 ** 40),
    (1, 300, 333, 32, 2 ** 30 - 1, True, FF, FF, None),
]


@pytest.mark.parametrize("H,Sq,Skv,buckets,reach,two,dtype,ttype,offset", BIAS)
def test_bias_alone(dev, H, Sq, Skv, buckets, reach, two, dtype, ttype, offset):
    g = torch.Generator().manual_seed(70)
    table = torch.randn(buckets, H, generator=g).to(ttype)
    t = table.to(dev).requires_grad_()
    near_offset = offset if offset is None or abs(offset) < 2 ** 31 else int(math.copysign(4 * reach + 4 * (Sq + Skv), offset))
    bucket = bucket_map(Sq, Skv, buckets, reach, two, near_offset)
    want = table[bucket].permute(2, 0, 1).to(dtype)
    out = cdna4_sage.relative_bias(t, Sq, Skv, two, reach, dtype, offset)
    assert out.is_contiguous() and torch.equal(out.cpu(), want)
    if offset is not None:
        for kind in ((torch.int64,) if abs(offset) >= 2 ** 31 else (torch.int64, torch.int32)):
            at = torch.tensor([offset], dtype=kind, device=dev)
            assert torch.equal(cdna4_sage.relative_bias(t, Sq, Skv, two, reach, dtype, at), out)
    # from gradients of every element, in all the shapes that they come in
    full = torch.randn(H, Sq, Skv, generator=g).to(dtype)
    for d in (full, full.transpose(1, 2).contiguous().transpose(1, 2), full[:1].expand(H, Sq, Skv), full[:, :1].expand(H, Sq, Skv),
              torch.ones((), dtype=dtype).expand(H, Sq, Skv)):
        got, = torch.autograd.grad(out, t, d.to(dev), retain_graph=True)
        x = d.double().reshape(H, -1).t()
        s, a = (torch.zeros(buckets, H, dtype=torch.float64).index_add_(0, bucket.flatten(), y.contiguous()) for y in (x, x.abs()))
        over = s.abs() > torch.finfo(ttype).max * (1 + half_step(ttype))      # (sums of ones pass fp16's largest number)
        assert bool(torch.isinf(got.cpu()[over]).all())
        got, s, a = (torch.where(over, 0.0, x.double().cpu()) for x in (got, s, a))
        # chunks of 64 rows, then at most 2 * 2048 / 64 + 8 diagonals a lane, in float32; the rest in float64
        close(got, s, half_step(ttype) * s.abs() + (64 + 128) * F32 * a)


def test_bias_of_more_rows_than_a_workgroup_has(dev):
    """Several chunks and segments; and a table that is a slice of a wider one."""
    H, Sq, Skv = 2, 700, 4500
    wide = torch.randn(32, 5, generator=torch.Generator().manual_seed(71)).to(dev).requires_grad_()
    t = wide[:, 1:3]
    out = cdna4_sage.relative_bias(t, Sq, Skv, dtype=BF)
    bucket = bucket_map(Sq, Skv, 32, 128, True)
    assert torch.equal(out.cpu(), t.detach().cpu()[bucket].permute(2, 0, 1).to(BF))
    d = _rand((H, Sq, Skv), 72)
    got, = torch.autograd.grad(out, wide, d.to(dev))
    x = d.double().reshape(H, -1).t()
    s, a = (torch.zeros(32, H, dtype=torch.float64).index_add_(0, bucket.flatten(), y.contiguous()) for y in (x, x.abs()))
    close(got[:, 1:3], s, (64 + 128 + 2) * F32 * a)
    assert bool((got[:, [0, 3, 4]] == 0).all())


def test_a_captured_token_moves_on(dev):
    table = _rand((32, 4), 73, FF).to(dev)
    at = torch.zeros(1, dtype=torch.int64, device=dev)
    cdna4_sage.relative_bias(table, 1, 500, False, q_offset=at)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cdna4_sage.relative_bias(table, 1, 500, False, q_offset=at)
    for p in (499, 0, 17, 250):
        at.fill_(p)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cdna4_sage.relative_bias(table, 1, 500, False, q_offset=p))


# ---- together -------------------------------------------------------------------------------------------------------------

def test_a_layer_is_trained_and_then_runs_quantized(dev):
    """Rotary positions, attention with a bias and its gradients through both, as a layer has them; then the trained layer's
    forward on the 8-bit attention with the bias as its mask."""
    B, H, Hkv, S, D = 1, 4, 2, 1100, 64
    g = torch.Generator().manual_seed(80)
    x = [torch.randn(B, h, S, D, generator=g).to(BF).to(dev).requires_grad_() for h in (H, Hkv, Hkv)]
    table = (torch.randn(32, H, generator=g) * 0.5).to(BF).to(dev).requires_grad_()
    do = _rand((B, H, S, D), 81).to(dev)
    freqs, factor = cdna4_sage.rope_frequencies(D, device=dev)
    q, k = cdna4_sage.rope(x[0], x[1], None, freqs, factor=factor)
    out = cdna4_sage.attention_train(q, k, x[2], bias_table=table)
    dq, dk, dv, dt = torch.autograd.grad(out, [*x, table], do)
    qs, ks = q.detach().requires_grad_(), k.detach().requires_grad_()
    part = cdna4_sage.attention_train(qs, ks, x[2], bias_table=table)
    assert torch.equal(part, out)
    aq, ak, av, at = torch.autograd.grad(part, [qs, ks, x[2], table], do)
    assert torch.equal(dv, av) and torch.equal(dt, at)
    back = torch.autograd.grad(cdna4_sage.rope(x[0], x[1], None, freqs, factor=factor), x[:2], (aq, ak))
    assert torch.equal(dq, back[0]) and torch.equal(dk, back[1])
    bucket = bucket_map(S, S, 32, 128, True)
    e = Exact(q.detach().cpu(), k.detach().cpu(), x[2].detach().cpu(), bias=table.detach().cpu().double()[bucket].permute(2, 0, 1),
              dout=do.cpu())
    close(out, e.out, e.room_out)
    close(aq, e.dq, e.room_dq)
    close(dt, *e.table(bucket, 32, bucket % 16 == 15, BF))
    with torch.no_grad():
        table -= 0.01 * dt
        bias = cdna4_sage.relative_bias(table, S, S)
        exact16 = cdna4_sage.attention_train(q, k, x[2], bias_table=table)
        quantized = cdna4_sage.attention(q.detach(), k.detach(), x[2].detach(), "HND", attn_mask=bias[None])
    a, b = exact16.double().flatten(), quantized.double().flatten()
    assert float((a @ b) / (a.norm() * b.norm())) > 0.995
