"""Decoder layers with e4m3 weights and a 4-bit paged cache, on the package's own operators.

    python examples/decoder_layer.py [--layers 2] [--hidden 5120] [--seqs 32] [--prompt 512] [--steps 16]

A layer is
    norm -> qkv -> rotation and append -> attention -> output projection
    + residual, norm -> silu(gate) * up -> down + residual
with every matrix product e4m3 x e4m3 (`fp8_linear.linear`), the norms and the
quantisation of activations in one pass each, and keys and values in 4.5 bits an
element (`kv4`).  Prompts and decode steps take the same path: a call has any
number of new tokens of any number of sequences.
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tans-vectoradd_b200"))

from rans_vectoradd import fp8_linear, kv4, tans_gemv  # noqa: E402


@dataclass
class Shape:
    hidden: int = 5120
    ffn: int = 17408
    q_heads: int = 40
    kv_heads: int = 8
    head_dim: int = 128
    page_size: int = 64


@dataclass
class Batch:
    """The new tokens of one call: which sequences hold them, and where they go."""
    positions: torch.Tensor  # int64 [tokens]
    slots: torch.Tensor      # int64 [tokens]
    table: torch.Tensor      # int32 [seqs, pages]
    lens: torch.Tensor       # int32 [seqs], the new tokens included
    starts: torch.Tensor     # int32 [seqs + 1]
    most_new: int


class Pages:
    """Page tables of a fixed set of sequences; pages are handed out in order."""

    def __init__(self, seqs: int, most: int, page_size: int, device):
        self.size, self.lens = page_size, [0] * seqs
        per = -(-most // page_size)
        self.pages = seqs * per
        self.table = torch.arange(self.pages, dtype=torch.int32, device=device).view(seqs, per)

    def extend(self, news: list[int]) -> Batch:
        """Room for news[b] more tokens of each sequence."""
        dev, T = self.table.device, sum(news)
        seq = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news))
        starts = torch.tensor([0] + news).cumsum(0)
        pos = torch.tensor(self.lens)[seq] + torch.arange(T) - starts[seq]
        self.lens = [a + b for a, b in zip(self.lens, news)]
        pos, seq = pos.to(dev), seq.to(dev)
        slots = self.table[seq, pos // self.size].long() * self.size + pos % self.size
        return Batch(pos, slots, self.table, torch.tensor(self.lens, dtype=torch.int32, device=dev),
                     starts.to(torch.int32).to(dev), max(news))


def rotation(shape: Shape, most: int, device, base: float = 10000.0):
    """cos and sin of each position, f32 [most, head_dim / 2]."""
    half = shape.head_dim // 2
    inv = base ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
    angle = torch.arange(most, device=device, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


class Layer:
    def __init__(self, shape: Shape, pages: int, device, generator: torch.Generator):
        self.shape = s = shape
        D = s.head_dim

        def weight(rows, cols):
            w = torch.randn(rows, cols, device=device, generator=generator) * cols ** -0.5
            return tans_gemv.quantize_rows(w)

        self.qkv = weight((s.q_heads + 2 * s.kv_heads) * D, s.hidden)
        self.out = weight(s.hidden, s.q_heads * D)
        self.gate, self.up = weight(s.ffn, s.hidden), weight(s.ffn, s.hidden)
        self.down = weight(s.hidden, s.ffn)
        one = lambda: (1 + 0.1 * torch.randn(s.hidden, device=device, generator=generator)).to(torch.bfloat16)  # noqa: E731
        self.norm1, self.norm2 = one(), one()
        self.cache = kv4.KV4Cache.allocate(pages, s.kv_heads, s.page_size, D, device)

    def __call__(self, h: torch.Tensor, b: Batch, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
        """h [tokens, hidden] bf16, the residual stream, after this layer."""
        s, T = self.shape, h.shape[0]
        D, nq, nk = s.head_dim, s.q_heads * s.head_dim, s.kv_heads * s.head_dim
        x8, xs, _ = fp8_linear.add_rms_norm_e4m3(h, self.norm1)
        qkv = fp8_linear.linear(x8, xs, *self.qkv)
        q, k, v = qkv[:, :nq].view(T, -1, D), qkv[:, nq:nq + nk].view(T, -1, D), qkv[:, nq + nk:].view(T, -1, D)
        q = kv4.append(self.cache, k, v, b.slots, positions=b.positions, cos=cos, sin=sin, q=q)
        a = kv4.attention(self.cache, q, b.table, b.lens, starts=b.starts, most_new=b.most_new)
        a8, a_s = fp8_linear.quantize_tokens(a.view(T, nq))
        o = fp8_linear.linear(a8, a_s, *self.out)
        x8, xs, h = fp8_linear.add_rms_norm_e4m3(o, self.norm2, h)
        up = fp8_linear.linear(x8, xs, *self.up)
        act = fp8_linear.linear(x8, xs, *self.gate, act="silu", mul=up, out=up)
        f8, fs = fp8_linear.quantize_tokens(act)
        return fp8_linear.linear(f8, fs, *self.down, residual=h)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("layers", 2), ("hidden", 5120), ("ffn", 17408), ("seqs", 32), ("prompt", 512), ("steps", 16)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(0)
    shape = Shape(hidden=a.hidden, ffn=a.ffn)
    most = a.prompt + a.steps
    pages = Pages(a.seqs, most, shape.page_size, dev)
    layers = [Layer(shape, pages.pages, dev, g) for _ in range(a.layers)]
    cos, sin = rotation(shape, most, dev)
    last = fp8_linear.add_rms_norm
    final = torch.ones(a.hidden, dtype=torch.bfloat16, device=dev)

    def run(news):
        b = pages.extend(news)
        h = torch.randn(sum(news), a.hidden, device=dev, generator=g).to(torch.bfloat16)
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ev[0].record()
        for layer in layers:
            h = layer(h, b, cos, sin)
        y, _ = last(h, final)
        ev[1].record()
        torch.cuda.synchronize()
        assert torch.isfinite(y).all()
        return ev[0].elapsed_time(ev[1])

    prompts = [max(1, a.prompt - 7 * i % a.prompt) for i in range(a.seqs)]
    ms = run(prompts)
    print(f"{sum(prompts)} prompt tokens of {a.seqs} sequences, {a.layers} layers: {ms:.2f} ms (first call)")
    times = sorted(run([1] * a.seqs) for _ in range(a.steps))
    print(f"decode step of {a.seqs} sequences: {times[len(times) // 2] / a.layers * 1e3:.0f} us a layer (median of {a.steps})")
    print(f"cache: {layers[0].cache.token_bytes()} bytes a token and layer")


if __name__ == "__main__":
    main()
