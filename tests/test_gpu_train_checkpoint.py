"""attention_train and relative_bias inside torch.utils.checkpoint, also where a dispatch mode is active, as under selective
checkpoints: what the backward pass needs is unpacked once."""
import pytest
import torch
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

import cdna4_sage

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _step(q, k, v, table, cu):
    out = cdna4_sage.attention_train(q, k, v, bias_table=table, is_causal=True)
    rows = [t[0].transpose(0, 1) for t in (q, k, v)]
    more = cdna4_sage.attention_train_varlen(*rows, cu, cu)
    bias = cdna4_sage.relative_bias(table, 9, 9, dtype=torch.float32)
    return out.float().square().sum() + more.float().square().sum() + bias.square().sum()


@pytest.mark.parametrize("how", ["plain", "recompute", "save"])
def test_checkpoints(dev, how):
    g = torch.Generator().manual_seed(81)
    q, k, v = (torch.randn(1, 4, 150, 64, generator=g).to(BF).to(dev) for _ in range(3))
    table = torch.randn(16, 4, generator=g).to(BF).to(dev)
    cu = torch.tensor([0, 60, 150], dtype=torch.int32, device=dev)

    def run(f):
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        return torch.autograd.grad(f(*leaves, cu), leaves)

    policy = {"recompute": CheckpointPolicy.PREFER_RECOMPUTE, "save": CheckpointPolicy.MUST_SAVE}
    more = {} if how == "plain" else {
        "context_fn": lambda: create_selective_checkpoint_contexts(lambda ctx, op, *args, **kwargs: policy[how])}
    want = run(_step)
    got = run(lambda *ts: checkpoint(_step, *ts, use_reentrant=False, **more))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
