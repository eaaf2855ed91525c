"""quantize_tokens is defined value by value: scale = max|x| / 448 (1 for a row of
zeros, at least the smallest normal f32) and q = e4m3(x / scale), each division
rounded once to f32 and the code to nearest even.  Codes and scales are compared for
equality with that, worked out on the CPU: no tolerance."""
from __future__ import annotations

import pytest
import torch

from rans_vectoradd import fp8_linear

LEAST = torch.tensor(2.0 ** -126)


def define(x):
    x = x.cpu().float()
    top = x.abs().amax(-1)
    scale = torch.where(top == 0, torch.ones_like(top), torch.maximum(top / torch.full_like(top, 448.0), LEAST))
    return (x / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def check(x):
    q, scale = fp8_linear.quantize_tokens(x)
    want_q, want_scale = define(x)
    assert torch.equal(scale.cpu(), want_scale)
    off = q.cpu() != want_q
    assert not off.any(), f"{int(off.sum())} of {off.numel()} codes differ"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(400, 5120), (3, 17408), (1, 1), (5, 255), (2000, 64), (300, 4099), (2, 32768),
                                       (2, 40000), (1, 57341)])
def test_codes_and_scales_are_the_definitions(cuda, dtype, rows, cols):
    g = torch.Generator(device=cuda).manual_seed(cols)
    x = torch.randn(rows, cols, device=cuda, generator=g)
    check(x.to(dtype))
    check((x * torch.exp2(torch.randint(-9, 9, (rows, 1), device=cuda, generator=g).float())).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows_at_any_address(cuda, dtype):
    g = torch.Generator(device=cuda).manual_seed(1)
    for cols in (256, 1023, 4100):
        for at in (0, 1, 3, 8):
            check(torch.randn(9, cols + 16, device=cuda, generator=g).to(dtype)[:, at:at + cols])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,least,most", [(torch.bfloat16, -133, 127), (torch.float16, -24, 15), (torch.float32, -149, 127)])
def test_sizes_to_the_ends_of_the_types(cuda, dtype, least, most):
    """Rows whose largest value is a power of two, from the smallest subnormal on, and a row of zeros."""
    g = torch.Generator().manual_seed(2)
    top = 2.0 ** torch.arange(least, most + 1).double()
    x = (torch.rand(len(top), 96, generator=g).double() * 2 - 1) * top[:, None]
    x[:, 0] = top
    x = torch.cat([x, torch.zeros(1, 96, dtype=torch.float64)]).to(dtype)
    check(x.to(cuda))
