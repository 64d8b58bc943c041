"""attention_train under torch.compile with lengths that change from call to call: one trace serves them all."""
import pytest
import torch
from torch._dynamo.testing import CompileCounterWithBackend

import cdna4_sage

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _run(f, ts, *rest):
    leaves = [t.clone().requires_grad_() for t in ts]
    out = f(*leaves, *rest)
    return (out, *torch.autograd.grad(out.float().square().sum(), leaves))


def _check(f, calls):
    torch._dynamo.reset()
    counter = CompileCounterWithBackend("aot_eager")
    compiled = torch.compile(f, backend=counter, fullgraph=True, dynamic=True)
    for ts, rest in calls:
        for a, b in zip(_run(f, ts, *rest), _run(compiled, ts, *rest)):
            assert torch.equal(a, b)
    assert counter.frame_count == 1
    torch._dynamo.reset()


def _draw(dev, seed, *shapes):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(BF).to(dev) for s in shapes]


def test_packed_totals(dev):
    def f(q, k, v, table, cu):
        return cdna4_sage.attention_train_varlen(q, k, v, cu, cu, is_causal=True, bias_table=table, bidirectional=False)

    calls = []
    for i, ends in enumerate(([30, 100], [64, 65, 200], [5, 9, 300, 517], [128, 256], [700, 701, 702, 1000], [2, 40])):
        n = ends[-1]
        calls.append((_draw(dev, i, (n, 4, 64), (n, 2, 64), (n, 2, 64), (16, 4)),
                      [torch.tensor([0, *ends], dtype=torch.int32, device=dev)]))
    _check(f, calls)


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_dense_lengths(dev, layout):
    def f(q, k, v, mask):
        return cdna4_sage.attention_train(q, k, v, layout, attn_mask=mask)

    calls = []
    # (the first call's batch is not the number of heads: torch takes sizes that are equal there for one symbol)
    for i, (B, Sq, Skv) in enumerate(((6, 70, 90), (3, 64, 200), (4, 333, 334), (2, 129, 65), (5, 20, 500))):
        shape = lambda H, S: (B, H, S, 128) if layout == "HND" else (B, S, H, 128)  # noqa: E731
        mask = torch.rand(B, 1, Sq, Skv, generator=torch.Generator().manual_seed(i)) < 0.6
        calls.append((_draw(dev, i, shape(4, Sq), shape(2, Skv), shape(2, Skv)), [mask.to(dev)]))
    _check(f, calls)
