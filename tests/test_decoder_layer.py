"""The example's decoder layers (examples/decoder_layer.py): prompts and decode
steps through the operators together, against the same layers in plain 64-bit
operations with the same roundings of what is stored (e4m3 activations, bf16
tensors, e2m1 cache).

The bound: two computations of a value that differ by bf16's rounding (2^-9 in
the mean) fall on different sides of an e4m3 step (2^-4 of it) once in 2^5 and
then differ by 2^-3: 2^-6 of its size in the mean.  A layer has four such roundings in
line on the way to its output and the cache's e2m1 (steps up to 2^-1, one in 2^7 on
different sides, 2^-5 in the mean) beside them, which the residual stream carries
on: at most 4 x 2^-6 + 2^-5 = 0.094 a layer of the layer's own part, and that is
under the stream's size.  Two layers: 0.19 at the worst, a tenth expected, as
the differences add like random ones."""
from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    m = importlib.util.module_from_spec(spec)
    import sys
    sys.modules["decoder_layer"] = m
    spec.loader.exec_module(m)
    return m


def bf(x):
    return x.to(torch.bfloat16).double()


def q8(x):
    """x as e4m3 with a scale a row, as values."""
    s = x.abs().amax(-1, keepdim=True).clamp_min(1e-300) / 448
    return (x / s).float().to(torch.float8_e4m3fn).double() * s


def matrix(w):
    return w[0].view(torch.float8_e4m3fn).double() * w[1].double()[:, None]


def norm(h, w):
    return h / (h.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()


def e2m1(x):
    b = x.unflatten(-1, (-1, 16))
    s = (b.abs().amax(-1, keepdim=True) / 6).float().to(torch.float8_e4m3fn).double()
    r = torch.where(s > 0, b / torch.where(s > 0, s, 1.0), 0.0).abs()
    step = torch.where(r < 2, 0.5, torch.where(r < 4, 1.0, 2.0))
    return (torch.sign(b) * (torch.round(r / step) * step).clamp(max=6.0) * s).flatten(-2)


def turn(x, cos, sin):
    a, b = x.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


class Plain:
    """A layer's parameters, keys and values per sequence."""

    def __init__(self, layer, seqs):
        self.l, self.held = layer, [([], []) for _ in range(seqs)]

    def __call__(self, h, b, cos, sin):
        L, s = self.l, self.l.shape
        T, D = h.shape[0], s.head_dim
        nq, nk, G = s.q_heads * D, s.kv_heads * D, s.q_heads // s.kv_heads
        qkv = bf(q8(norm(h, L.norm1)) @ matrix(L.qkv).t())
        c, n = cos[b.positions], sin[b.positions]
        q = bf(turn(qkv[:, :nq].view(T, -1, D), c, n))
        k = e2m1(turn(qkv[:, nq:nq + nk].view(T, -1, D), c, n))
        v = e2m1(qkv[:, nq + nk:].view(T, -1, D))
        out = []
        starts = b.starts.tolist()
        for i, (keys, vals) in enumerate(self.held):
            lo, hi = starts[i], starts[i + 1]
            keys.append(k[lo:hi])
            vals.append(v[lo:hi])
            K, V = torch.cat(keys).repeat_interleave(G, 1), torch.cat(vals).repeat_interleave(G, 1)
            score = torch.einsum("thd,lhd->thl", q[lo:hi], K) / math.sqrt(D)
            last = K.shape[0] - (hi - lo) + torch.arange(hi - lo, device=h.device)
            hidden = torch.arange(K.shape[0], device=h.device)[None] > last[:, None]
            out.append(torch.einsum("thl,lhd->thd", score.masked_fill(hidden[:, None], -math.inf).softmax(-1), V))
        a = bf(torch.cat(out)).reshape(T, nq)
        o = bf(q8(a) @ matrix(L.out).t())
        x8 = q8(norm(o + h, L.norm2))
        h = bf(o + h)
        up = bf(x8 @ matrix(L.up).t())
        g = x8 @ matrix(L.gate).t()
        act = bf(g * torch.sigmoid(g) * up)
        return bf(q8(act) @ matrix(L.down).t() + h)


@pytest.mark.gpu
@pytest.mark.parametrize("page_size,head_dim,kv_heads", [(16, 64, 2), (64, 128, 1)])
def test_layers_against_plain_operations(cuda, page_size, head_dim, kv_heads):
    m = example()
    g = torch.Generator(device=cuda).manual_seed(page_size)
    shape = m.Shape(hidden=512, ffn=1040, q_heads=4, kv_heads=kv_heads, head_dim=head_dim, page_size=page_size)
    prompts = [33, 1, 70]
    pages = m.Pages(3, 100, page_size, cuda)
    layers = [m.Layer(shape, pages.pages, cuda, g) for _ in range(2)]
    plain = [Plain(layer, 3) for layer in layers]
    cos, sin = m.rotation(shape, 100, cuda)
    for news in (prompts, [1, 1, 1], [3, 1, 2], [1, 1, 1]):
        b = pages.extend(news)
        x = torch.randn(sum(news), 512, device=cuda, generator=g).to(torch.bfloat16)
        h, want = x, x.double()
        for layer, p in zip(layers, plain):
            h, want = layer(h, b, cos, sin), p(want, b, cos, sin)
        err = float((h.double() - want).norm() / want.norm())
        assert err <= 0.19, err
        assert not torch.equal(h, x)


@pytest.mark.gpu
def test_decode_one_by_one_equals_all_at_once(cuda):
    """Tokens appended and attended one a call see the same cache as in one call: the same rows but for the
    order of sums."""
    m = example()
    shape = m.Shape(hidden=256, ffn=512, q_heads=4, kv_heads=2, head_dim=64, page_size=16)
    outs = []
    for split in (False, True):
        g = torch.Generator(device=cuda).manual_seed(1)
        pages = m.Pages(2, 40, 16, cuda)
        layer = m.Layer(shape, pages.pages, cuda, g)
        cos, sin = m.rotation(shape, 40, cuda)
        x = torch.randn(2, 5, 256, device=cuda, generator=g).to(torch.bfloat16)
        if split:
            rows = [layer(x[:, i].contiguous(), pages.extend([1, 1]), cos, sin) for i in range(5)]
            outs.append(torch.stack(rows, 1))
        else:
            outs.append(layer(x.reshape(10, 256), pages.extend([5, 5]), cos, sin).view(2, 5, 256))
    a, b = (o.double() for o in outs)
    assert float((a - b).norm() / b.norm()) <= 4 * 2.0 ** -6
