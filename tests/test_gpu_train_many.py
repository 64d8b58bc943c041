"""attention_train over thousands of short sequences, dense and packed."""
import pytest
import torch

import cdna4_sage
from test_gpu_train import _compare, _draw, _run
from train_util import Exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,H,Hkv,S,D,dtype", [(8192, 16, 4, 3, 64, torch.bfloat16), (4500, 16, 16, 2, 64, torch.float16)])
def test_many_entries(dev, B, H, Hkv, S, D, dtype):
    q, k, v, do = _draw(B, H, Hkv, S, S, D, dtype, seed=61)
    e = Exact(q, k, v, causal=True, dout=do)
    _compare(e, *_run(dev, q, k, v, do, is_causal=True))

    # the same one behind the other
    rows = [t.transpose(1, 2).flatten(0, 1).to(dev).requires_grad_() for t in (q, k, v)]
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev) * S
    out, lse = cdna4_sage.attention_train_varlen(*rows, cu, cu, is_causal=True, return_lse=True)
    grads = torch.autograd.grad(out, rows, do.transpose(1, 2).flatten(0, 1).to(dev))
    back = lambda t: t.unflatten(0, (B, S)).transpose(1, 2)  # noqa: E731
    _compare(e, back(out), lse.unflatten(1, (B, S)).transpose(0, 1), [back(t) for t in grads])
