"""cdna4_sage.rope on the GPU under forward-mode derivatives and torch.func's transforms: the rotation is linear, so tangents
are the turned tangents bit for bit, and mapped calls what the entries give alone."""
import pytest
import torch
from torch.autograd import forward_ad

import cdna4_sage

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout, interleaved, dtype", [("NHD", False, torch.bfloat16), ("HND", True, torch.float16)])
def test_transforms(dev, layout, interleaved, dtype):
    B, S, H, Hk, D = 2, 9, 4, 2, 64
    g = torch.Generator().manual_seed(1)

    def new(h, *lead):
        x = torch.randn(*lead, B, S, h, D, generator=g).to(dtype).to(dev)
        return x if layout == "NHD" else x.transpose(-3, -2).contiguous()

    q, k, tq, tk = new(H), new(Hk), new(H), new(Hk)
    freqs = cdna4_sage.rope_frequencies(32)[0].to(dev)
    pos = torch.arange(B * S, device=dev).view(B, S) * 111
    f = lambda a, b: cdna4_sage.rope(a, b, pos, freqs, layout, interleaved, 1.25)  # noqa: E731
    one = lambda a: cdna4_sage.rope(a, None, pos, freqs, layout, interleaved, 1.25)  # noqa: E731
    want, turned = f(q, k), f(tq, tk)
    out, tangent = torch.func.jvp(f, (q, k), (tq, tk))
    for a, b in zip((*out, *tangent), (*want, *turned)):
        assert torch.equal(a, b)
    for flag in (False, True):
        with forward_ad.dual_level():
            a, b = f(forward_ad.make_dual(q.clone().requires_grad_(flag), tq), k)
            assert torch.equal(forward_ad.unpack_dual(a).tangent, turned[0])
            t = forward_ad.unpack_dual(b).tangent
            assert t is None or not bool(t.any())
    x = q.clone().requires_grad_(True)
    (back,) = torch.autograd.grad(one(x), x, tq)
    assert torch.equal(torch.func.vjp(one, q)[1](tq)[0], back)
    many = new(H, 5)
    each = torch.stack([one(y) for y in many])
    assert torch.equal(torch.vmap(one)(many), each)
    assert torch.equal(torch.vmap(one, in_dims=2)(many.movedim(0, 2)), each)
    a, b = torch.vmap(f, in_dims=(0, None))(many, k)
    assert torch.equal(a, each) and torch.equal(b, want[1].expand_as(b))
    per = torch.arange(5 * S, device=dev).view(5, S)
    got = torch.vmap(lambda y, p: cdna4_sage.rope(y, None, p, freqs, layout, interleaved))(many, per)
    assert torch.equal(got, torch.stack([cdna4_sage.rope(y, None, p, freqs, layout, interleaved) for y, p in zip(many, per)]))


def test_traced_with_head_dim_outside(dev):
    """Inputs and gradients whose memory order has another dimension innermost, against the eager call."""
    g = torch.Generator().manual_seed(2)
    q, k, dq = (torch.randn(2, h, 64, 16, generator=g).half().to(dev).transpose(2, 3) for h in (4, 2, 4))
    freqs = cdna4_sage.rope_frequencies(64)[0].to(dev)
    want = cdna4_sage.rope(q.contiguous(), k.contiguous(), None, freqs)
    fn = torch.compile(lambda a, b: [y * 1.0 for y in cdna4_sage.rope(a, b, None, freqs)], backend="aot_eager", fullgraph=True)
    for got in (fn(q, k), cdna4_sage.rope(q, k, None, freqs)):
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    torch.library.opcheck(torch.ops.cdna4_sage.rope_qk.default, (q, k, None, freqs, "HND", False, 1.0, False),
                          test_utils=("test_schema", "test_faketensor"))
    x = q.detach().requires_grad_(True)
    (a,) = torch.autograd.grad(fn(x, k)[0], x, dq)
    y = q.contiguous().requires_grad_(True)
    (b,) = torch.autograd.grad(cdna4_sage.rope(y, None, None, freqs), y, dq.contiguous())
    assert torch.equal(a, b)
