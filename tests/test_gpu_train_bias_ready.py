"""attention_train with a bias inside where a workgroup has one or two tiles of keys, whose loads cover least of the time in which the
bias' values come to LDS: every wave has to wait for all of them."""
import pytest
import torch

from test_gpu_train import _compare, _draw, _run
from train_util import Exact, bucket_map, close

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("D,dtype,Sq,Skv", [(64, BF, 128, 30), (128, HF, 1, 64), (96, BF, 700, 65), (256, HF, 128, 64)])
def test_values_of_the_farthest_reach_over_few_keys(dev, D, dtype, Sq, Skv):
    """1521 values a head, of which each query takes those of the other end."""
    B, H, buckets, far = 16, 4, 256, 790
    q, k, v, do = _draw(B, H, H, Sq, Skv, D, dtype, seed=91)
    table = (torch.randn(buckets, H, generator=torch.Generator().manual_seed(92)) * 2).to(dtype)
    bucket = bucket_map(Sq, Skv, buckets, far, True)
    e = Exact(q, k, v, bias=table.double()[bucket].permute(2, 0, 1), dout=do)
    first = _run(dev, q, k, v, do, table=table, max_distance=far)
    for _ in range(3):
        out, lse, grads = _run(dev, q, k, v, do, table=table, max_distance=far)
        _compare(e, out, lse, grads[:3])
        close(grads[3], *e.table(bucket, buckets, bucket % 128 == 127, dtype))
        assert torch.equal(out, first[0]) and all(torch.equal(a, b) for a, b in zip(grads, first[2]))
