"""Attention over the 4-bit cache where most of a row's keys weigh little beside a
few: every 32nd key has score 18 and value 0, all others score 0 and value 1, so
the output is the share of e^-18 = 2^-26 weights and nothing else.

A weight enters the second product in f16 relative to 2^-7 of the row's largest: it errs by at
most 2^-32 of that, in a sum of at least one such weight a peak.  Besides, u|o| for
the output's rounding (u = 2^-8 bf16, 2^-11 f16, 2^-25 where f16 is subnormal), 2^-11 |o| for
the weights above f16's subnormals, and the scores' own error e = (dim + 16) 2^-23 18 + 2^-20 (18 + 1),
which moves a weight by e of itself."""
from __future__ import annotations

import math

import pytest
import torch

from rans_vectoradd import kv4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 64])
@pytest.mark.parametrize("keys,group", [(500, 4), (9000, 4), (500, 16), (40000, 9)])
def test_small_weights_count(cuda, dtype, dim, page, keys, group):
    pages = -(-keys // page)
    cache = kv4.KV4Cache.allocate(pages, 1, page, dim, cuda)
    cache.k_scales.fill_(0x38)  # 1
    cache.v_scales.fill_(0x38)
    peak = (torch.arange(pages * page, device=cuda) % 32 == 0).view(pages, page)
    cache.k_codes[:, 0, :, 0] = torch.where(peak, 7, 0).to(torch.uint8)  # element 0: 6 or 0
    cache.v_codes[:, 0] = torch.where(peak, 0, 0x22)[:, :, None].to(torch.uint8)  # all elements 0 or 1
    q = torch.zeros(1, group, dim, device=cuda, dtype=dtype)
    q[:, :, 0] = 3.0
    out, lse = kv4.attention(cache, q, torch.arange(pages, dtype=torch.int32, device=cuda)[None],
                             torch.tensor([keys], dtype=torch.int32, device=cuda), scale=1.0, return_lse=True)
    peaks = -(-keys // 32)
    low = (keys - peaks) * math.exp(-18)
    want, e = low / (peaks + low), (dim + 16) * 2.0 ** -23 * 18 + 2.0 ** -20 * 19
    u, tiny = (2.0 ** -8, 0.0) if dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -25)
    bound = 1.01 * u * want + tiny + (2.0 ** -11 + 2 * e + 2.0 ** -18) * want + keys * 2.0 ** -32 / peaks
    off = float((out.double() - want).abs().max())
    assert off <= bound, f"{off / bound} of the bound, {off / want} of the output"
    lse_off = float((lse.double() - (18 + math.log(peaks + low))).abs().max())
    assert lse_off <= e + 2.0 ** -18 + 2.0 ** -21 * (18 + math.log(peaks + low))
