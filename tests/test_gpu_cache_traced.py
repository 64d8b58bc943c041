"""The cache's ops under tracers in both layouts: what their fake implementations promise, and the same bits as eager calls."""
import pytest
import torch

import cdna4_sage
from cache_util import as_int8, random_cache
from test_gpu_cache import _to, _tree

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("code", [torch.int8, E4M3])
def test_traced_in_both_layouts(dev, layout, code):
    g = torch.Generator().manual_seed(15)
    B, T, H, Hkv, D, n = 2, 3, 4, 2, 96, 16
    lengths = torch.tensor([20, 9], dtype=torch.int32, device=dev)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    base = _to(dev, random_cache(g, 4, n, Hkv, D, code))
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(torch.bfloat16).to(dev) for h in (H, Hkv, Hkv))
    if layout == "HND":
        q, k, v = (t.transpose(1, 2).contiguous() for t in (q, k, v))
    slots, tree = cdna4_sage.cache_slots(table, lengths, T, n), _tree(g, B, T).to(dev)
    freqs = cdna4_sage.rope_frequencies(32)[0].to(dev)

    def fn(q, k, v, *cache):
        cache = cdna4_sage.KVCache(*cache)
        out = cdna4_sage.cache_step(q, k, v, cache, slots, table, lengths, freqs=freqs, tensor_layout=layout)
        again, lse = cdna4_sage.cache_attention(q, cache, table, lengths, layout, tree_mask=tree, return_lse=True)
        return (out * 1.0, again.flatten(0, 1) * 1.0, lse, *(t * 1.0 for t in cdna4_sage.cache_read(cache, slots, torch.float16, layout)))

    c1, c2 = (tuple(t.clone() for t in base) for _ in range(2))
    want = fn(q, k, v, *c1)
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(q, k, v, *c2)
    for a, b in zip(want, got):
        assert torch.equal(a, b) and a.stride() == b.stride()
    for a, b in zip(c1, c2):
        assert torch.equal(as_int8(a) if a.dim() == 4 else a, as_int8(b) if b.dim() == 4 else b)
    # (torch's schema check multiplies its inputs, which it cannot for E4M3)
    tests = ("test_schema", "test_faketensor") if code == torch.int8 else ("test_faketensor",)
    ops = torch.ops.cdna4_sage
    for mask in (None, tree):
        for op in (ops.cache_attention.default, ops.cache_attention_lse.default):
            torch.library.opcheck(op, (q, *base, table, lengths, mask, layout, 0.0, True), test_utils=tests)
    torch.library.opcheck(ops.cache_read.default, (*base, slots, torch.bfloat16, layout), test_utils=("test_faketensor",))


def test_what_the_kernels_do_not_address_is_unsupported(dev):
    """Cache tensors off 16-byte boundaries and masks of far strides are refused as what the kernel does not take, not by an
    error of the library."""
    cache = cdna4_sage.new_cache(2, 16, 2, 64, device=dev)
    q, x = torch.zeros(1, 4, 3, 64, dtype=torch.float16, device=dev), torch.zeros(3, 2, 64, dtype=torch.float16, device=dev)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    slots = torch.zeros(3, dtype=torch.int64, device=dev)
    for name in cdna4_sage.KVCache._fields:
        t = getattr(cache, name)
        odd = torch.zeros(t.numel() + 2, dtype=t.dtype, device=dev)[2:].view(t.shape)
        assert odd.is_contiguous() and odd.data_ptr() % 16
        bad = cache._replace(**{name: odd})
        for call in (lambda: cdna4_sage.cache_attention(q, bad, table, lengths), lambda: cdna4_sage.cache_read(bad, slots),
                     lambda: cdna4_sage.cache_write(bad, x, x, slots)):
            with pytest.raises(cdna4_sage.Unsupported):
                call()
    far = torch.empty(2**30 + 16, dtype=torch.bool, device=dev)
    for strides in ((2**29, 1), (1, 2**29)):
        with pytest.raises(cdna4_sage.Unsupported):
            cdna4_sage.cache_attention(q, cache, table, lengths, tree_mask=far.as_strided((3, 3), strides))
    one = far.as_strided((1, 1), (2**40, 2**40))                  # (a single token's mask takes no stride)
    assert not bool(cdna4_sage.cache_attention(q[:, :, :1], cache, table, lengths, tree_mask=one).any())
