"""The decoding operators under forward-mode derivatives, torch.func's transforms and mixed gradient flags, without a GPU:
rope's launch is replaced by the rotation in torch, so that what is tested is how its derivatives are put together."""
import pytest
import torch
from torch.autograd import forward_ad

import cdna4_sage
from cache_util import rotate
from cdna4_sage import _rope

F = cdna4_sage.rope_frequencies(8)[0]
B, S, H, D = 2, 3, 4, 16


@pytest.fixture(autouse=True)
def turned_by_torch(monkeypatch):
    def launch(q, k, positions, freqs, layout, interleaved, factor, inverse):
        def turn(x):
            if x is None:
                return None
            assert layout == "NHD" and x.dim() == 4
            x.data_ptr()     # (a transform's wrapper has none)
            pos = torch.arange(x.shape[1]) if positions is None else positions
            return rotate(x.double(), pos.expand(x.shape[:2]), freqs, interleaved, factor, inverse)[0].to(x.dtype)

        return turn(q), turn(k)

    monkeypatch.setattr(_rope, "rope_launch", launch)


def _r(seed, *shape):
    return torch.randn(*(shape or (B, S, H, D)), generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


POS = torch.tensor([[5, 900, 31], [7, 0, 12]])


def _rope1(x, freqs=F, positions=POS):
    return cdna4_sage.rope(x, None, positions, freqs, "NHD", factor=1.5)


def _rope2(x, y):
    return cdna4_sage.rope(x, y, POS, F, "NHD", True, 1.5)


def _turn(x, interleaved=False, back=False, freqs=F, positions=POS):
    return rotate(x, positions, freqs, interleaved, 1.5, back)[0]


def _same(a, b):
    assert a.shape == b.shape and torch.allclose(a, b, rtol=1e-13, atol=1e-13)


@pytest.mark.parametrize("grad", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("tangents", [(True, False), (False, True), (True, True)])
def test_tangents_turn_as_the_inputs_do(grad, tangents):
    q, k, tq, tk = _r(1).requires_grad_(grad[0]), _r(2).requires_grad_(grad[1]), _r(3), _r(4)
    with forward_ad.dual_level():
        a = forward_ad.make_dual(q, tq) if tangents[0] else q
        b = forward_ad.make_dual(k, tk) if tangents[1] else k
        for got, t, has in zip(_rope2(a, b), (tq, tk), tangents):
            got = forward_ad.unpack_dual(got).tangent
            _same(torch.zeros_like(t) if got is None else got, _turn(t, True) if has else torch.zeros_like(t))
        if tangents[0]:
            _same(forward_ad.unpack_dual(_rope1(a)).tangent, _turn(tq))


def test_torch_func():
    q, t = _r(5), _r(6)
    out, tangent = torch.func.jvp(_rope1, (q,), (t,))
    _same(out, _turn(q)), _same(tangent, _turn(t))
    tq, tk = torch.func.jvp(lambda x: _rope2(x, q), (q,), (t,))[1]
    _same(tq, _turn(t, True))
    assert not bool(tk.any())
    _same(torch.func.grad(lambda x: (_rope1(x) * t).sum())(q), _turn(t, back=True))
    # |R x|^2 = 1.5^2 |x|^2 over the turned channels: its second derivative along t is 2 * 1.5^2 t there, 2 t elsewhere
    want = 2 * torch.cat([2.25 * t[..., :8], t[..., 8:]], -1)
    square = lambda x: (_rope1(x) ** 2).sum()  # noqa: E731
    _same(torch.func.jvp(torch.func.grad(square), (q,), (t,))[1], want)
    _same(torch.func.grad(lambda x: torch.func.jvp(square, (x,), (t,))[1])(q), want)
    _same(torch.func.grad(lambda x: (torch.func.grad(square)(x) * t).sum())(q), want)
    _same(torch.func.jacfwd(_rope1)(q).flatten(4).flatten(0, 3) @ t.flatten(), _turn(t).flatten())
    _same(torch.func.jacrev(_rope1)(q).flatten(4).flatten(0, 3) @ t.flatten(), _turn(t).flatten())


def test_vmap():
    x = _r(7, 5, B, S, H, D)
    want = torch.stack([_turn(y) for y in x])
    _same(torch.vmap(_rope1)(x), want)
    _same(torch.vmap(_rope1, in_dims=3, out_dims=2)(x.movedim(0, 3)), want.movedim(0, 2))
    _same(torch.vmap(torch.vmap(_rope1))(x.expand(2, 5, B, S, H, D)), want.expand(2, 5, B, S, H, D))
    _same(torch.vmap(torch.func.grad(lambda y, u: (_rope1(y) * u).sum()))(x, x), torch.stack([_turn(y, back=True) for y in x]))
    _same(torch.vmap(lambda y, u: torch.func.jvp(_rope1, (y,), (u,))[1])(x, x), want)
    q, k = torch.vmap(_rope2, in_dims=(0, None))(x, x[0])
    _same(q, torch.stack([_turn(y, True) for y in x])), _same(k, _turn(x[0], True).expand_as(x))
    # positions and frequencies of each entry's own, shared ones of the three shapes
    pos = torch.arange(5 * B * S).view(5, B, S)
    _same(torch.vmap(lambda p: _rope1(x[0], positions=p))(pos), torch.stack([_turn(x[0], positions=p) for p in pos]))
    for p in (pos[0, :1], pos[0, 0], None):
        full = (torch.arange(S) if p is None else p).expand(B, S)
        _same(torch.vmap(lambda y: _rope1(y, positions=p))(x), torch.stack([_turn(y, positions=full) for y in x]))
    _same(torch.vmap(lambda p: _rope1(x[0], positions=p), in_dims=1)(pos[0].t()),
          torch.stack([_turn(x[0], positions=p.expand(B, S)) for p in pos[0]]))
    fs = torch.stack([F, F * 2])
    _same(torch.vmap(lambda f: _rope1(x[0], f))(fs), torch.stack([_turn(x[0], freqs=f) for f in fs]))
    q, k = torch.vmap(lambda f: cdna4_sage.rope(x[0], x[1], POS, f, "NHD", factor=1.5))(fs)
    _same(k, torch.stack([_turn(x[1], freqs=f) for f in fs]))
    with pytest.raises(cdna4_sage.Unsupported):
        torch.vmap(lambda p: _rope1(x[0], positions=p))(pos[:, :1].expand(5, 3, S))


def test_a_tracer_refuses_tangents():
    q, t = _r(8), _r(9)
    compiled = torch.compile(lambda x, u: torch.func.jvp(_rope1, (x,), (u,))[1], backend="aot_eager")
    _same(compiled(q, t), _turn(t))       # (the tracer leaves the call to eager execution)
    torch._dynamo.reset()
    with pytest.raises(Exception):
        torch.compile(lambda x, u: torch.func.jvp(_rope1, (x,), (u,))[1], backend="aot_eager", fullgraph=True)(q, t)


# ---- the cache's operators, which have no derivative ------------------------------------------------------------------

def _attend(monkeypatch, read=False):
    """cache_attention (or cache_read) of q and the scales with its launch replaced by a product."""
    from cdna4_sage import _cache

    def launch(q, cache, table, lengths, layout, *rest):
        q.data_ptr()
        return q * cache.k_scale.sum(), None

    monkeypatch.setattr(_cache, "attention_launch", launch)
    monkeypatch.setattr(_cache, "read_launch", lambda cache, slots, dtype, layout: (cache.k_scale * 2, cache.v_scale * 2))
    cache = cdna4_sage.new_cache(2, 16, 2, 64, device="cpu")
    table, lengths, slots = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    if read:
        return lambda _, scale: cdna4_sage.cache_read(cache._replace(k_scale=scale), slots)[0], cache
    return lambda q, scale: cdna4_sage.cache_attention(q, cache._replace(k_scale=scale), table, lengths, "NHD"), cache


@pytest.mark.parametrize("read", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_the_cache_refuses_tangents(monkeypatch, read, grad):
    call, cache = _attend(monkeypatch, read)
    q, s = torch.randn(1, 1, 4, 64), cache.k_scale + 1
    call(q, s)
    with forward_ad.dual_level():
        call(q, s)                                            # no tangent: as ever
        with pytest.raises(NotImplementedError):
            call(q, forward_ad.make_dual(s.clone().requires_grad_(grad), s))
        if not read:
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(q.clone().requires_grad_(grad), q), s)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: call(q, x), (s,), (s,))
    with pytest.raises(NotImplementedError):
        torch.vmap(lambda x, u: torch.func.jvp(lambda y: call(q, y), (x,), (u,))[1])(s[None], s[None])
    # (one of the transformed function's constants has none)
    out, tangent = torch.func.jvp(lambda x: x * call(q, s).sum(), (s,), (s,))
    assert torch.equal(out, tangent)


def test_only_outputs_of_inputs_that_need_a_gradient_need_one():
    for flags in ((True, False), (False, True), (True, True), (False, False)):
        q, k = (_r(10 + i).requires_grad_(flag) for i, flag in enumerate(flags))
        out = _rope2(q, k)
        assert tuple(y.requires_grad for y in out) == flags
        if not any(flags):
            continue
        got = torch.autograd.grad([y for y in out if y.requires_grad], [x for x in (q, k) if x.requires_grad],
                                  [_r(20 + i) for i in range(sum(flags))], create_graph=True)
        for i, x in enumerate(got):
            _same(x, _turn(_r(20 + i), True, back=True))
    with torch.no_grad():
        assert not any(y.requires_grad for y in _rope2(_r(1).requires_grad_(True), _r(2)))
    # (a gradient of a gradient in one of two)
    q, k = _r(11).requires_grad_(True), _r(12)
    u = _r(13).requires_grad_(True)
    (g,) = torch.autograd.grad(_rope2(q, k)[0], q, u, create_graph=True)
    (gg,) = torch.autograd.grad(g, u, _r(14))
    _same(gg, _turn(_r(14), True))


# ---- what tracers are told about the outputs --------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_rope_outputs_have_the_strides_that_tracers_are_told(monkeypatch, layout):
    from torch._subclasses.fake_tensor import FakeTensorMode

    monkeypatch.undo()                         # the launch itself, without its kernel
    monkeypatch.setattr(_rope._capi, "call_on", lambda *a: None)

    def check(q, k, positions, freqs, layout):
        b, s, h, d = q.shape if layout == "NHD" else (q.shape[0], q.shape[2], q.shape[1], q.shape[3])
        return b, s, h, d, 0

    monkeypatch.setattr(_rope, "check_rope", check)
    base = torch.zeros(2, 8, 16, 64, dtype=torch.float16)
    forms = [base, base.transpose(1, 2), base.permute(0, 1, 3, 2).contiguous().transpose(2, 3),
             base.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0), torch.zeros(0, 8, 16, 64, dtype=torch.float16), base[:, :, :1].expand(2, 8, 16, 64),
             torch.zeros(2, 8, 16, 65, dtype=torch.float16)[..., :64], base[:1],
             torch.zeros(12345 + 8192, dtype=torch.float16).as_strided((1, 8, 16, 64), (12345, 1024, 64, 1))]
    f = cdna4_sage.rope_frequencies(64)[0]
    for x in forms:
        real = torch.ops.cdna4_sage.rope_qk(x, x, None, f, layout, False, 1.0, False)
        one = torch.ops.cdna4_sage.rope(x, None, f, layout, False, 1.0, False)
        with FakeTensorMode() as mode:
            y = mode.from_tensor(x)
            fake = torch.ops.cdna4_sage.rope_qk(y, y, None, mode.from_tensor(f), layout, False, 1.0, False)
            only = torch.ops.cdna4_sage.rope(y, None, mode.from_tensor(f), layout, False, 1.0, False)
        for a, b in zip((*real, one), (*fake, only)):
            assert a.shape == b.shape and a.stride() == b.stride(), x.stride()
