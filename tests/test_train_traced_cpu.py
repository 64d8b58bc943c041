"""attention_train under a tracer with symbolic sizes: the fake op ties no length down, and its state is as large as the library's."""
import random

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import cdna4_sage
from cdna4_sage import _capi

pytestmark = pytest.mark.skipif(not _capi.LIB_PATH.exists(), reason="libsage_capi.so not built")


def _leaves(*shapes):
    return [torch.zeros(s, dtype=torch.bfloat16, requires_grad=True) for s in shapes]


def _dense(mask, bias):
    def fn(q, k, v, table, m):
        out = cdna4_sage.attention_train(q, k, v, attn_mask=m if mask else None, bias_table=table if bias else None)
        return torch.autograd.grad(out.sum(), (q, k, v))
    return fn


def _packed(q, k, v, cu):
    out = cdna4_sage.attention_train_varlen(q, k, v, cu, cu)
    return torch.autograd.grad(out.sum(), (q, k, v))


def _state_of(graph):
    node, = [n for n in graph.graph.nodes if n.target == torch.ops.cdna4_sage.attention_train.default]
    return node.meta["val"][2].shape[0]


@pytest.mark.parametrize("mask,bias", [(False, False), (True, False), (False, True), (True, True)])
def test_dense_lengths_stay_symbols(mask, bias):
    args = (*_leaves((3, 4, 70, 64), (3, 2, 90, 64), (3, 2, 90, 64)), torch.zeros(32, 4), torch.ones(3, 1, 70, 90, dtype=torch.bool))
    graph = make_fx(_dense(mask, bias), tracing_mode="symbolic")(*args)
    n = _state_of(graph)
    assert isinstance(n, torch.SymInt)
    q, k = [p.meta["val"] for p in graph.graph.nodes if p.op == "placeholder"][:2]
    assert all(isinstance(x, torch.SymInt) and x.node.expr.free_symbols for x in (q.shape[0], q.shape[2], k.shape[2]))
    assert q.shape[2].node.expr.free_symbols <= n.node.expr.free_symbols


def test_packed_totals_stay_symbols():
    args = (*_leaves((130, 4, 64), (140, 2, 64), (140, 2, 64)), torch.tensor([0, 30, 100, 130], dtype=torch.int32))
    graph = make_fx(_packed, tracing_mode="symbolic")(*args)
    q, k, _, cu = [p.meta["val"] for p in graph.graph.nodes if p.op == "placeholder"]
    want = set().union(*(x.node.expr.free_symbols for x in (q.shape[0], k.shape[0], cu.shape[0])))
    assert len(want) == 3 and want <= _state_of(graph).node.expr.free_symbols


def test_the_state_is_as_large_as_the_library_says():
    rng = random.Random(5)
    size = lambda top: int(2 ** rng.uniform(0, top))  # noqa: E731
    fake = torch._subclasses.FakeTensorMode
    for i in range(300):
        packed, keep, D = rng.random() < 0.3, rng.random() < 0.7, rng.choice((64, 96, 128, 256))
        B, Hkv, Sq, Skv = size(5), size(3), size(13), size(13)
        H = Hkv * size(2)
        bias = (32, rng.random() < 0.5, rng.choice((100, 300, 700))) if rng.random() < 0.4 else None
        mask = None if packed or rng.random() < 0.5 else tuple(rng.choice((1, n)) for n in (B, H, Sq, Skv))
        with fake():
            e = lambda *s: torch.empty(*s, dtype=torch.bfloat16)  # noqa: E731
            table = None if bias is None else torch.empty(bias[0], H)
            m = None if mask is None else torch.empty(mask, dtype=torch.bool)
            how = (0.0, False, True if bias is None else bias[1], 128 if bias is None else bias[2], keep)
            op = torch.ops.cdna4_sage.attention_train
            if packed:
                cu = torch.empty(B + 1, dtype=torch.int32)
                got = op(e(Sq, H, D), e(Skv, Hkv, D), e(Skv, Hkv, D), None, table, cu, cu, "NHD", *how)[2].shape[0]
            elif i % 2:
                got = op(e(B, Sq, H, D), e(B, Skv, Hkv, D), e(B, Skv, Hkv, D), m, table, None, None, "NHD", *how)[2].shape[0]
            else:
                got = op(e(B, H, Sq, D), e(B, Hkv, Skv, D), e(B, Hkv, Skv, D), m, table, None, None, "HND", *how)[2].shape[0]
        axes = None if mask is None else tuple(int(n > 1) for n in mask[:3])
        assert got == _capi.train_workspace(packed, B, H, Hkv, Sq, Skv, D, axes, bias, keep)[0], (packed, B, H, Sq, Skv, D, mask, bias)
