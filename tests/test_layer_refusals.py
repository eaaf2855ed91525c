"""Arrays off their elements' alignment, and sums whose rows overlap, are refused by the
decoder-layer entry points before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

from rans_vectoradd import fp8_linear
from rans_vectoradd._lib import KV4, LIB

P = 256  # an aligned address that is never followed


def refused(rc, word):
    assert rc == 1 and word in LIB.tans_b200_last_error().decode(), (rc, LIB.tans_b200_last_error())


def test_norm_alignment():
    def norm(x=P, r=P, w=P, wt=0, h=P, y=None, q=P, s=P, rows=2, hs=8, dt=0):
        return LIB.tans_b200_add_rms_norm(x, 8, r, 8, w, wt, 1e-6, h, hs, y, q, s, rows, 8, dt, None)
    for kw in ({"x": P + 1}, {"r": P + 1}, {"w": P + 1}, {"h": P + 1}, {"s": P + 2}, {"y": P + 1, "q": None, "s": None},
               {"x": P + 2, "dt": 2, "wt": 2}, {"w": P + 2, "wt": 2}):
        refused(norm(**kw), "aligned")
    for hs in (0, 1, 7, -7):
        refused(norm(hs=hs), "overlap")
    refused(LIB.tans_b200_quantize_tokens(P + 1, 8, P, P, 1, 8, 0, None), "aligned")
    refused(LIB.tans_b200_quantize_tokens(P, 8, P, P + 2, 1, 8, 0, None), "aligned")


def test_linear_alignment():
    def linear(xs=P, ws=P, b=P, mul=P, r=P, y=P, status=P):
        return LIB.tans_b200_linear(P, xs, P, ws, b, 0, mul, r, y, 1, 8, 16, 0, status, None)
    for kw in ({"xs": P + 2}, {"ws": P + 2}, {"b": P + 1}, {"mul": P + 1}, {"r": P + 1}, {"y": P + 1}, {"status": P + 2}):
        refused(linear(**kw), "aligned")


def test_kv4_alignment():
    def cache(**kw):
        f = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, k_gain=None, v_gain=None, pages=4, heads=2, page_size=16, dim=128)
        f.update(kw)
        return ctypes.byref(KV4(*f.values()))

    def append(c=None, slots=P, pos=P, status=P):
        return LIB.tans_b200_kv4_append(c or cache(), P, 256, P, 256, slots, None, 0, 0, None, pos, P, P, 10, 8, 0, 1, 0, status, None)

    def read(c=None, slots=P, status=P):
        return LIB.tans_b200_kv4_read(c or cache(), slots, P, P, 1, 0, status, None)

    def attend(c=None, table=P, lens=P, starts=P, lse=P, status=P):
        return LIB.tans_b200_kv4_attention(c or cache(), P, 512, 4, table, 4, 4, lens, starts, 1, 1, 1, 1.0, 0, P, lse, P, 1 << 30, 0,
                                           status, None)
    for call in (append, read, attend):
        for kw in ({"k_gain": P + 2}, {"v_gain": P + 1}):
            refused(call(cache(**kw)), "aligned")
        refused(call(status=P + 2), "aligned")
    for kw in ({"slots": P + 4}, {"pos": P + 4}):
        refused(append(**kw), "aligned")
    refused(read(slots=P + 4), "aligned")
    for kw in ({"table": P + 2}, {"lens": P + 2}, {"starts": P + 1}, {"lse": P + 2}):
        refused(attend(**kw), "aligned")


@pytest.mark.gpu
def test_a_sum_in_the_place_of_a_broadcast_input_is_refused(cuda):
    x, w = torch.randn(4, 64, device=cuda), torch.ones(64, device=cuda)
    r = torch.randn(1, 64, device=cuda).expand(4, 64)
    keep = r.clone()
    with pytest.raises(RuntimeError, match="overlap"):
        fp8_linear.add_rms_norm(x, w, r, residual_out=r)
    with pytest.raises(RuntimeError, match="overlap"):
        fp8_linear.add_rms_norm_e4m3(x, w, r, residual_out=torch.empty(64 + 3 * 8, device=cuda).as_strided((4, 64), (8, 1)))
    assert torch.equal(r, keep)
    y, h = fp8_linear.add_rms_norm(x, w, r)
    assert torch.equal(h, x + r) and torch.isfinite(y).all()
    one = r[:1]
    fp8_linear.add_rms_norm(x[:1], w, one, residual_out=one)
    assert torch.equal(one, x[:1] + keep[:1])
