"""A caller's workspace for attention over the 4-bit cache: used when it fits, refused by
the Python call when it is no contiguous uint8 tensor of the device or too small."""
from __future__ import annotations

import pytest
import torch

from rans_vectoradd import kv4


@pytest.mark.gpu
def test_workspaces(cuda):
    cache = kv4.KV4Cache.allocate(64, 2, 16, 64, cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.random_(0, 256)
    for t in (cache.k_scales, cache.v_scales):
        t.fill_(0x30)
    q = torch.randn(1, 4, 64, device=cuda).to(torch.bfloat16)
    table, lens = torch.arange(64, dtype=torch.int32, device=cuda)[None], torch.tensor([1000], dtype=torch.int32, device=cuda)
    need = kv4.attention_workspace_bytes(2, 16, 64, 4, 64, 1, 1, 1, 0, cuda)
    assert need
    call = lambda ws: kv4.attention(cache, q, table, lens, workspace=ws)  # noqa: E731
    want = call(None)
    assert torch.equal(call(torch.empty(need, dtype=torch.uint8, device=cuda)), want)
    assert torch.equal(call(torch.empty(need + 64, dtype=torch.uint8, device=cuda)[16:-48]), want)
    for bad in (torch.empty(need, dtype=torch.uint8), torch.empty(2 * need, dtype=torch.uint8, device=cuda)[::2],
                torch.empty(need, dtype=torch.float32, device=cuda), torch.empty(need - 1, dtype=torch.uint8, device=cuda),
                torch.empty(need + 1, dtype=torch.uint8, device=cuda)[1:], torch.empty(1, dtype=torch.uint8, device=cuda).expand(need)):
        with pytest.raises(RuntimeError):
            call(bad)
    assert torch.equal(call(None), want)
    # a call that needs none still looks at what it is given
    short = torch.tensor([16], dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError):
        kv4.attention(cache, q, table[:, :1], short, workspace=torch.empty(need, dtype=torch.uint8))
