"""attention_train at the ends of sm_scale's range: outputs and gradients, or a refusal, never gradients of 0."""
import pytest
import torch

import cdna4_sage
from test_gpu_train import _compare, _draw, _run
from train_util import Exact

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, BF), (256, BF)])
@pytest.mark.parametrize("sm_scale", [2.0 ** -100, 2.0 ** -60])
def test_small_ones(dev, D, dtype, sm_scale):
    """All weights alike: the gradient of the values is what is left."""
    q, k, v, do = _draw(1, 2, 2, 130, 300, D, dtype, seed=71)
    out, lse, grads = _run(dev, q, k, v, do, sm_scale=sm_scale)
    e = Exact(q, k, v, dout=do, sm_scale=sm_scale)
    _compare(e, out, lse, grads)
    assert bool((grads[2] != 0).any())


def test_scores_of_ordinary_size_from_large_inputs(dev):
    q, k, v, do = _draw(1, 2, 1, 100, 150, 64, BF, seed=73)
    q, k = (t.float() * 2.0 ** 48 for t in (q, k))
    q, k = q.to(BF), k.to(BF)
    out, lse, grads = _run(dev, q, k, v, do, sm_scale=2.0 ** -99)
    e = Exact(q, k, v, dout=do, sm_scale=2.0 ** -99)
    _compare(e, out, lse, grads)


def test_the_largest(dev):
    q, k, v, do = _draw(1, 1, 1, 70, 90, 64, BF, seed=75)
    q, k = ((t.float() * 2.0 ** -65).to(BF) for t in (q, k))
    q[:, :, 3] = 0.0
    out, lse, grads = _run(dev, q, k, v, do, sm_scale=2.0 ** 127)
    e = Exact(q, k, v, dout=do, sm_scale=2.0 ** 127)
    _compare(e, out, lse, grads)


def test_beyond(dev):
    q, k, v, _ = (t.to(dev) for t in _draw(1, 1, 1, 20, 20, 64, BF))
    leaf = q.clone().requires_grad_()
    for sm_scale in (2.0 ** -101, 2.0 ** -126):
        with pytest.raises(cdna4_sage.Unsupported, match="sm_scale"):
            cdna4_sage.attention_train(leaf, k, v, sm_scale=sm_scale)
        # without a backward pass it is a mean
        out = cdna4_sage.attention_train(q, k, v, sm_scale=sm_scale)
        mean = v.double().mean(2, keepdim=True).expand_as(out)
        assert float((out.double() - mean).abs().max()) <= 2.0 ** -7 * float(v.double().abs().mean())
    for sm_scale in (2.0 ** 127.5, 3.4e38):
        with pytest.raises(cdna4_sage.Unsupported, match="sm_scale"):
            cdna4_sage.attention_train(q, k, v, sm_scale=sm_scale)
