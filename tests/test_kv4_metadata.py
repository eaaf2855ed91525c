"""Attention over the 4-bit cache when `starts` is malformed: the rows of a
refused sequence are zeros with lse -inf, whatever the output's memory held,
and the other sequences' rows are as without it."""
from __future__ import annotations

import pytest
import torch

from rans_vectoradd import _C, kv4


def setup(dev, columns, page=16):
    """Three sequences of 70, 33 and 40 tokens in a table of `columns` pages at most, and 7 queries."""
    g = torch.Generator(device=dev).manual_seed(columns)
    cache = kv4.KV4Cache.allocate(16, 2, page, 128, dev)
    for t in (cache.k_codes, cache.v_codes):
        t.copy_(torch.randint(0, 256, t.shape, device=dev, generator=g, dtype=torch.uint8))
    for t in (cache.k_scales, cache.v_scales):
        t.copy_(torch.randint(0x20, 0x38, t.shape, device=dev, generator=g, dtype=torch.uint8))
    table = torch.zeros(3, columns, dtype=torch.int32, device=dev)
    for b, (at, n) in enumerate(((0, 5), (5, 3), (8, 3))):
        table[b, :n] = torch.arange(at, at + n)
    q = torch.randn(7, 6, 128, device=dev, generator=g).to(torch.bfloat16)
    return cache, q, table, torch.tensor([70, 33, 40], dtype=torch.int32, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [20, 300])  # too few pages at most to split the keys, and enough
@pytest.mark.parametrize("starts,most_new,good", [
    ([0, 2, 3, 7], 3, [0, 1]),          # the last has four
    ([0, 2, 3, 7], None, [1]),          # one a sequence without most_new
    ([0, 3, 4, 7], 2, [1]),             # the first and the last have three
    ([-2, 1, 3, 7], 4, [1, 2]),         # begins before q
    ([0, 2, 5, 9], 4, [0, 1]),          # ends after it
    ([2, 4, 2 ** 31 - 1, 2 ** 31 - 1], 2, [0]),
    ([-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1], 7, []),
    ([1, 2, 3, 2], 1, [0, 1])])         # descends
def test_rows_of_refused_sequences_are_zeros(cuda, columns, starts, most_new, good):
    cache, q, table, lens = setup(cuda, columns)
    want, want_lse = torch.zeros_like(q), torch.full((7, 6), float("-inf"), device=cuda)
    for b in good:
        rows = slice(starts[b], starts[b + 1])
        n = starts[b + 1] - starts[b]
        want[rows], want_lse[rows] = kv4.attention(
            cache, q[rows], table[b:b + 1], lens[b:b + 1], starts=torch.tensor([0, n], dtype=torch.int32, device=cuda),
            most_new=n, return_lse=True)
    kw = {} if most_new is None else {"most_new": most_new}
    # a row of a sequence that lies after the last start as well may be either
    keep = [i for i in range(7) if starts[3] >= starts[2] or i != 2]
    # what the outputs' memory may hold
    torch.full((7, 6, 128), float("nan"), dtype=torch.bfloat16, device=cuda)
    torch.full((7, 6), float("nan"), device=cuda)
    _C.data_status()
    got, lse = kv4.attention(cache, q, table, lens, starts=torch.tensor(starts, dtype=torch.int32, device=cuda),
                             return_lse=True, **kw)
    assert _C.data_status() == 16
    spare = [i for i in keep if not want[i].any()]
    assert not got[spare].any() and torch.isneginf(lse[spare]).all()
    # other parts of the keys may be summed first where the batch splits them otherwise
    assert torch.allclose(got[keep].float(), want[keep].float(), rtol=2.0 ** -7, atol=2.0 ** -9)
    fin = torch.isfinite(want_lse[keep])
    assert torch.allclose(lse[keep][fin], want_lse[keep][fin], rtol=2.0 ** -16, atol=2.0 ** -14)
