"""What append stores at the edges of rounding, for keys and for values, code by code:
ties, saturation, zeros of either sign, infinities and NaN.  The cache's bytes are
defined bit by bit, so nothing here has a tolerance."""
from __future__ import annotations

import pytest
import torch

from rans_vectoradd import kv4
from test_kv4 import angles, gen, rotate32, to_codes


def edges():
    x = torch.zeros(1, 1, 128)
    x[0, 0, :16] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6])
    x[0, 0, 16:19] = torch.tensor([6.375, -0.0, 1.0])   # scale 1.0625, half way between 1 and 1.125
    x[0, 0, 32:34] = torch.tensor([2.0 ** -8 * 6, -2.0 ** -14])  # a subnormal scale; a value that rounds to -0
    x[0, 0, 48:50] = torch.tensor([2.0 ** -12, -2.0 ** -12])     # the scale rounds to 0
    x[0, 0, 64:66] = torch.tensor([30000.0, -5000.0])            # past the largest scale
    x[0, 0, 80], x[0, 0, 96], x[0, 0, 112] = float("inf"), float("nan"), -float("inf")
    return x


def held(cache, slots):
    """Codes one a byte, and scales, of the tokens in the given slots."""
    page = cache.page_size
    at = (slots // page, slice(None), slots % page)
    out = []
    for n in "kv":
        c = getattr(cache, n + "_codes").cpu()[at]
        out += [torch.stack([c & 15, c >> 4], -1).flatten(-2), getattr(cache, n + "_scales").cpu()[at]]
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rounding_edges_of_keys_and_values(cuda, dtype):
    x = edges().to(dtype)
    cache = kv4.KV4Cache.allocate(1, 1, 1, 128, cuda)
    slot = torch.zeros(1, dtype=torch.int64, device=cuda)
    kv4.append(cache, x.to(cuda), x.to(cuda), slot)
    for r in kv4.read(cache, slot, torch.float32):
        r = r.cpu()[0, 0]
        assert r[:16].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, -6]
        assert r[16] == 6.0 and r[17] == 0 and r[18] == 1.0
        assert r[32] == 2.0 ** -8 * 6 and r[33] == 0 and not r[48:64].any()
        assert r[64] == 448 * 6 and r[65] == -448 * 6 and not r[66:80].any()
        assert r[80] == 448 * 6 and not r[81:96].any()
        assert torch.isnan(r[96:112]).all()
        assert r[112] == -448 * 6 and not r[113:].any()
    kc, ks, vc, vs = held(cache, torch.zeros(1, dtype=torch.int64))
    assert torch.equal(kc, vc) and torch.equal(ks, vs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,half,interleaved", [(64, 32, False), (128, 64, True), (128, 13, False), (256, 0, False)])
def test_codes_differ_at_most_in_the_sign_of_a_zero(cuda, dtype, dim, half, interleaved):
    T, H, page = 50, 3, 16
    g = gen(dim + half)
    k, v = (torch.randn(T, H, dim, generator=g).to(dtype) for _ in "kv")
    v[::7] = 0
    v[1::7, :, ::3] = -0.0
    slots = torch.randperm(5 * page, generator=g)[:T]
    pos = torch.randint(0, 500, (T,), generator=g)
    cos, sin = angles(500, half)
    cache = kv4.KV4Cache.allocate(5, H, page, dim, cuda)
    rot = dict(positions=pos.to(cuda), cos=cos.to(cuda), sin=sin.to(cuda)) if half else {}
    kv4.append(cache, k.to(cuda), v.to(cuda), slots.to(cuda), interleaved=interleaved, **rot)
    kc, ks, vc, vs = held(cache, slots)
    turned = rotate32(k.float(), cos[pos], sin[pos], interleaved) if half else k.float()
    for got, got_scales, x in ((kc, ks, turned), (vc, vs, v.float())):
        packed, scales = to_codes(x)
        want = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
        assert torch.equal(got_scales, scales)
        off = got != want
        assert not ((got & 7)[off]).any() and not ((want & 7)[off]).any()
        assert torch.equal(got & 7, want & 7)
