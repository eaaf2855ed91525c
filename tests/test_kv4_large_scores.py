"""Attention over the 4-bit cache with scores so large that f32 holds them in steps of
8 to 2048 (in base 2): all values are 1, so whatever the weights, the output is 1 and
the lse lies between the largest score and that of all keys together."""
from __future__ import annotations

import math

import pytest
import torch

from rans_vectoradd import kv4


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("keys,group", [(256, 4), (256, 16), (2000, 4)])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores_weigh_finitely(cuda, dim, keys, group, sign):
    page = 32
    pages = -(-keys // page)
    cache = kv4.KV4Cache.allocate(pages, 1, page, dim, cuda)
    cache.k_scales.fill_(0x38)  # 1
    cache.v_scales.fill_(0x38)
    cache.v_codes.fill_(0x22)
    # element 0 of every key: 1; element 1: 0, then 0.5 .. 6 in later keys of each warp
    step = (torch.arange(pages * page, device=cuda) // 128 % 8).view(pages, page)
    cache.k_codes[:, 0, :, 0] = (2 + 16 * step).to(torch.uint8)
    sizes = [(k, d) for k in range(22, 35) for d in (1.0, 2.0, 4.0, 8.0, 16.0, 24.0, 32.0, 64.0)]
    q = torch.zeros(len(sizes), group, dim)
    for i, (k, d) in enumerate(sizes):
        q[i, :, 0], q[i, :, 1] = sign * 2.0 ** k, d
    q = q.to(torch.bfloat16)
    n = len(sizes)
    table = torch.arange(pages, dtype=torch.int32, device=cuda).expand(n, pages)
    out, lse = kv4.attention(cache, q.to(cuda), table, torch.full((n,), keys, dtype=torch.int32, device=cuda),
                             scale=math.log(2), return_lse=True)
    assert torch.equal(out, torch.ones_like(out))
    held = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=cuda, dtype=torch.float64)[step.flatten()[:keys]]
    x = q[:, 0].to(cuda).double()
    top = ((x[:, :1] + x[:, 1:2] * held) * math.log(2)).amax(1)
    slack = 2.0 ** -21 * top.abs()  # the score, its factor and the sum of maximum and logarithm, each rounded in f32
    lse = lse.double()
    assert bool((lse >= (top - slack - 1e-3)[:, None]).all()) and bool((lse <= (top + slack + math.log(keys) + 1e-3)[:, None]).all())
