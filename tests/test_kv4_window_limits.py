"""A window of any size up to 2^63 - 1 (a caller's "no limit") takes the launch form
and the workspace of a call without one, and gives its result."""
from __future__ import annotations

import pytest
import torch

from rans_vectoradd import kv4


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1 << 20, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 62, 2 ** 63 - 2, 2 ** 63 - 1])
def test_huge_windows_are_none(cuda, window):
    cache = kv4.KV4Cache.allocate(64, 2, 64, 64, cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.random_(0, 256)
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(0x30)
    sizes = (2, 64, 64, 4, 64, 1, 3, 3)
    assert kv4.attention_workspace_bytes(*sizes, window, cuda) == kv4.attention_workspace_bytes(*sizes, 0, cuda) > 0
    q = torch.randn(3, 4, 64, device=cuda).to(torch.bfloat16)
    table, lens = torch.arange(64, dtype=torch.int32, device=cuda)[None], torch.tensor([4000], dtype=torch.int32, device=cuda)
    call = lambda w: kv4.attention(cache, q, table, lens, starts=torch.tensor([0, 3], dtype=torch.int32, device=cuda),  # noqa: E731
                                   most_new=3, window=w)
    assert torch.equal(call(window), call(0))
