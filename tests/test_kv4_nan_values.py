"""A NaN among the values of a key that a row sees makes the row's elements NaN, as
0 * NaN does in the formula, wherever the key lies: also where its weight is 0 in f32
and its warp, its part of the keys or its page is another than the largest score's."""
from __future__ import annotations

import pytest
import torch

from rans_vectoradd import kv4


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("keys,group,page", [(300, 4, 16), (300, 16, 64), (12000, 4, 32), (3000, 3, 8)])
def test_a_nan_of_no_weight_counts(cuda, dim, keys, group, page):
    pages = -(-keys // page)
    cache = kv4.KV4Cache.allocate(pages, 1, page, dim, cuda)
    cache.k_scales.fill_(0x38)  # 1
    cache.v_scales.fill_(0x38)
    cache.v_codes.fill_(0x22)   # 1
    at = lambda key: (key // page, 0, key % page)  # noqa: E731
    cache.k_codes[at(5)][0] = 7  # element 0: 6, a score of 6000; all others 0
    q = torch.zeros(1, group, dim, device=cuda, dtype=torch.bfloat16)
    q[:, :, 0] = 1000.0
    args = (q, torch.arange(pages, dtype=torch.int32, device=cuda)[None], torch.tensor([keys], dtype=torch.int32, device=cuda))
    assert torch.equal(kv4.attention(cache, *args, scale=1.0), torch.ones_like(q))
    for key in {0, 7, 40, 130, 299, keys // 2, keys - 1}:
        cache.v_scales[at(key)][1] = 0x7F
        out, lse = kv4.attention(cache, *args, scale=1.0, return_lse=True)
        cache.v_scales[at(key)][1] = 0x38
        assert torch.isnan(out[..., 16:32]).all(), key
        assert bool((out[..., :16] == 1).all()) and bool((out[..., 32:] == 1).all()) and bool(((lse - 6000).abs() < 0.01).all())
