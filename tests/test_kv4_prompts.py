"""Attention of a prompt's tokens over the 4-bit cache: hundreds of tiles a head, new
tokens alone and after held ones, against 64 bits within the bounds of test_kv4."""
from __future__ import annotations

import pytest
import torch

from test_kv4 import check_attention


@pytest.mark.gpu
@pytest.mark.parametrize("dim,lens,news,heads,group,page,window,dtype", [
    (64, [1300], [1300], 1, 4, 16, 0, torch.bfloat16),              # a prompt from its start
    (128, [2050, 1100, 1], [1021, 1100, 1], 1, 4, 64, 0, torch.bfloat16),  # beside a decode step, and after held tokens
    (64, [1500, 700], [1100, 699], 2, 5, 32, 300, torch.float16),   # within a window
    (128, [1200], [1200], 1, 7, 8, 0, torch.float16),               # pages shorter than a copy
    (256, [1030], [1030], 1, 2, 16, 0, torch.bfloat16),
    (64, [600] * 4, [600] * 4, 1, 1, 128, 0, torch.bfloat16)])
def test_prompts(cuda, dim, lens, news, heads, group, page, window, dtype):
    check_attention(cuda, lens, news, heads, group, dim, page, dtype, window=window, seed=dim + group)
