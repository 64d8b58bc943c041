"""cache_attention at the ends of its range: tiny and infinite queries, values of very different sizes side by side, places
that a row does not see, and the joining of many rows that come in several parts each."""
import pytest
import torch

from cache_util import random_cache
from test_gpu_cache import _compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, D", [(1, 64), (2, 128), (24, 96), (20, 256), (44, 128)])
@pytest.mark.parametrize("high", [0, 1, 2, 3])
def test_neighbouring_tiles_of_very_different_values(dev, rows, D, high):
    """One tile of 32 keys in four has values of 2^93, the others of 2^-86, with scores alike: each wave has a reference of its
    own, 2^179 apart, and the sums have to come together all the same."""
    g = torch.Generator().manual_seed(rows + high)
    page, n = 32, 256 - 7
    cache = list(random_cache(g, 8, page, 1, D, torch.int8))
    tile = torch.arange(8).view(8, 1, 1) % 4
    cache[3] = torch.where(tile == high, 2.0**86, 2.0**-93) * (1 + torch.rand(8, 1, page, generator=g))
    q = torch.randn(1, rows, 1, D, generator=g).to(torch.bfloat16)
    table, lengths = torch.arange(8, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    _compare(dev, q, cache, table, lengths)
    cache[3] = torch.where(tile == high, 2.0**-93, 2.0**86) * (1 + torch.rand(8, 1, page, generator=g))
    _compare(dev, q, cache, table, lengths)
