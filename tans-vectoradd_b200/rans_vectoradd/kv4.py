"""Keys and values in a paged 4-bit cache (no counterpart in the reference).

The cache of a decoder whose weights are this package's e4m3: 16 elements of a
head are 8 bytes of e2m1 codes and one e4m3 scale, 4.5 bits an element, and an
element is code * scale * gain[head].  `append` rotates and stores new tokens
(and rotates their queries in the same launch), `read` gives stored tokens
back, `attention` runs new tokens over the cache.  All of it on sm_100a kernels
(csrc/kv4.cu), on torch's current stream.

    cache = kv4.KV4Cache.allocate(pages, kv_heads, page_size=64, head_dim=128, device="cuda")
    q = kv4.append(cache, k, v, slots, positions=pos, cos=cos, sin=sin, q=q)
    out = kv4.attention(cache, q, block_table, lens)

Slots, positions, pages and lengths are device data: what is out of range is
never followed and shows in `rans_vectoradd._C.data_status()` (bit 16).
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from ._C import _post_check, _req, _status
from ._lib import LIB, KV4, check, on_device, ptr, raw_stream

_HALF = {torch.bfloat16: 0, torch.float16: 1}
_FLOAT = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@dataclass(init=False)
class KV4Cache:
    """k/v codes u8 [pages, heads, page_size, dim/2] and e4m3 scales u8
    [pages, heads, page_size, dim/16]; optional f32 gains [heads].  A field may be
    set to another tensor that fits the rest (gains found after the cache was
    made), which the next call then uses; other shapes need another cache."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    k_gain: torch.Tensor | None = None
    v_gain: torch.Tensor | None = None

    def __init__(self, k_codes, k_scales, v_codes, v_scales, k_gain=None, v_gain=None):
        self._bind(k_codes, k_scales, v_codes, v_scales, k_gain, v_gain)

    def _bind(self, kc, ks, vc, vs, kg, vg):
        """Checks the fields and takes them, with what the calls pass of them, all or none."""
        shape, u8 = kc.shape, torch.uint8
        if len(shape) != 4 or shape[3] not in (32, 64, 128):
            raise RuntimeError("codes must be [pages, heads, page_size, dim/2] with dim 64, 128 or 256")
        pages, heads, size, half = shape
        if size < 1 or size & (size - 1):
            raise RuntimeError("page_size must be a power of two")
        dev, scales = kc.device, (pages, heads, size, half // 8)
        if (not kc.is_cuda or vc.shape != shape or ks.shape != scales or vs.shape != scales
                or kc.dtype != u8 or vc.dtype != u8 or ks.dtype != u8 or vs.dtype != u8
                or vc.device != dev or ks.device != dev or vs.device != dev
                or not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous())):
            raise RuntimeError("cache arrays must be contiguous CUDA uint8, codes [.., dim/2] and scales [.., dim/16], "
                               "on one device")
        for t in (kg, vg):
            if t is not None:
                _req(t.dtype == torch.float32 and t.shape == (heads,) and t.is_contiguous() and t.device == dev,
                     "gains must be contiguous f32 [heads]")
        c = KV4(kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), ptr(kg), ptr(vg), pages, heads, size, 2 * half)
        # (_dev and so on: what every call asks for; a ctypes field takes longer to read)
        self.__dict__.update(k_codes=kc, k_scales=ks, v_codes=vc, v_scales=vs, k_gain=kg, v_gain=vg,
                             _c=c, _ref=ctypes.addressof(c), _dev=dev, _kv_heads=heads, _page=size, _dim=2 * half)

    def __setattr__(self, name: str, value) -> None:
        fields = self.__dataclass_fields__
        if name in fields:
            self._bind(*(value if f == name else getattr(self, f) for f in fields))
        else:
            object.__setattr__(self, name, value)

    def __delattr__(self, name: str) -> None:
        if name in self.__dataclass_fields__:
            raise AttributeError(f"{name} cannot be deleted; gains may be set to None")
        object.__delattr__(self, name)

    @classmethod
    def allocate(cls, pages: int, heads: int, page_size: int = 64, head_dim: int = 128,
                 device="cuda", k_gain=None, v_gain=None) -> "KV4Cache":
        """A cache of zeros."""
        z = lambda per: torch.zeros(pages, heads, page_size, head_dim // per,  # noqa: E731
                                    dtype=torch.uint8, device=device)
        return cls(z(2), z(16), z(2), z(16), k_gain, v_gain)

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    @property
    def heads(self) -> int:
        return self._c.heads

    @property
    def page_size(self) -> int:
        return self._c.page_size

    @property
    def head_dim(self) -> int:
        return self._c.dim

    def token_bytes(self) -> int:
        """Bytes that one token takes, keys and values of all heads."""
        return self.heads * self.head_dim * 9 // 8


def _heads(name: str, t: torch.Tensor, dim: int, dtype: torch.dtype, dev: torch.device) -> tuple[int, int, int]:
    """Checks [tokens, heads, dim] with dense heads: (tokens, heads, stride between tokens)."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or t.dtype != dtype or t.device != dev:
        raise RuntimeError(f"{name} must be [tokens, heads, {dim}] {dtype} on the cache's device")
    n, heads, _ = shape
    if t.is_contiguous():
        return n, heads, heads * dim
    st = t.stride()
    if st[2] != 1 or (st[1] != dim and heads != 1):
        raise RuntimeError(f"{name}'s heads must be dense (strides {dim} and 1)")
    return n, heads, st[0] if n > 1 else heads * dim


def _index(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, dev: torch.device) -> int:
    if t.dtype != dtype or t.shape != (n,) or not t.is_contiguous() or t.device != dev:
        raise RuntimeError(f"{name} must be a contiguous {dtype} tensor of {n} on the cache's device")
    return t.data_ptr()


def append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, *,
           positions: torch.Tensor | None = None, cos: torch.Tensor | None = None,
           sin: torch.Tensor | None = None, q: torch.Tensor | None = None,
           interleaved: bool = False) -> torch.Tensor | None:
    """Store tokens k, v [tokens, heads, dim] (bf16 or f16) in slots [tokens]
    int64 (page * page_size + place; negative: not stored; no two alike), the
    keys rotated by positions [tokens] int64, rows of cos and sin f32
    [max_position, half] (pairs (i, i + half), or (2i, 2i+1) if interleaved;
    2 * half <= dim).  Returns q [tokens, q_heads, dim] rotated alike, if given."""
    dt, dev, dim = k.dtype, cache._dev, cache._dim
    if dt not in _HALF:
        raise RuntimeError("k must be bfloat16 or float16")
    T, heads, ks = _heads("k", k, dim, dt, dev)
    vt, vheads, vs = _heads("v", v, dim, dt, dev)
    if heads != cache._kv_heads or vheads != heads or vt != T:
        raise RuntimeError("k and v must have the cache's heads")
    half = top = qs = qh = 0
    pos_p = cos_p = sin_p = q_p = out = out_p = None
    if positions is not None:
        if cos is None or sin is None:
            raise RuntimeError("positions need cos and sin")
        shape, f32 = cos.shape, torch.float32
        if (len(shape) != 2 or sin.shape != shape or cos.dtype != f32 or sin.dtype != f32 or not cos.is_contiguous()
                or not sin.is_contiguous() or cos.device != dev or sin.device != dev):
            raise RuntimeError("cos and sin must be contiguous f32 [max_position, half] on the cache's device")
        top, half = shape
        pos_p, cos_p, sin_p = _index("positions", positions, T, torch.int64, dev), cos.data_ptr(), sin.data_ptr()
    elif cos is not None or sin is not None:
        raise RuntimeError("cos and sin need positions")
    slots_p = _index("slots", slots, T, torch.int64, dev)
    with on_device(dev):
        if q is not None:
            qt, qh, qs = _heads("q", q, dim, dt, dev)
            if qt != T:
                raise RuntimeError("q must have k's tokens")
            q_p, out = q.data_ptr(), torch.empty(T, qh, dim, dtype=dt, device=dev)
            out_p = out.data_ptr()
        check(LIB.tans_b200_kv4_append(
            cache._ref, k.data_ptr(), ks, v.data_ptr(), vs, slots_p, q_p, qs, qh, out_p, pos_p, cos_p,
            sin_p, top, half, interleaved, T, _HALF[dt], _status(dev).data_ptr(), raw_stream(dev)))
    _post_check(dev)
    return out


def read(cache: KV4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
         ) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values [tokens, heads, dim] that the cache holds in slots
    [tokens] int64 (zeros for a negative slot)."""
    _req(dtype in _FLOAT, "dtype must be bfloat16, float16 or float32")
    dev, T = cache._dev, slots.shape[0]
    with on_device(dev):
        k = torch.empty(T, cache._kv_heads, cache._dim, dtype=dtype, device=dev)
        v = torch.empty_like(k)
        check(LIB.tans_b200_kv4_read(cache._ref, _index("slots", slots, T, torch.int64, dev), k.data_ptr(),
                                     v.data_ptr(), T, _FLOAT[dtype], _status(dev).data_ptr(), raw_stream(dev)))
    _post_check(dev)
    return k, v


@functools.lru_cache(maxsize=4096)
def attention_workspace_bytes(heads: int, page_size: int, head_dim: int, q_heads: int, max_pages: int, seqs: int,
                              tokens: int, most_new: int, window: int, device: torch.device) -> int:
    """Bytes of `attention`'s workspace: it follows from the sizes and the device alone."""
    c, n = KV4(256, 256, 256, 256, None, None, 1, heads, page_size, head_dim), ctypes.c_int64()
    with on_device(device):
        check(LIB.tans_b200_kv4_attention_workspace_bytes(ctypes.addressof(c), q_heads, max_pages, seqs, tokens,
                                                          most_new, window, ctypes.byref(n)))
    return n.value


def attention(cache: KV4Cache, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
              starts: torch.Tensor | None = None, most_new: int = 1, scale: float | None = None,
              window: int = 0, return_lse: bool = False, workspace: torch.Tensor | None = None):
    """out [tokens, q_heads, dim] of new tokens q over the cache.

    table [seqs, max_pages] int32: the pages of each sequence; lens [seqs]
    int32: the tokens it holds, its new ones (already appended) last.  starts
    [seqs + 1] int32: the rows of q that are each sequence's new tokens, at
    most most_new of them; without it every sequence has one.  Causal: the i-th
    of n new tokens sees keys up to lens - n + i, only the last `window` of them
    if window > 0.  scale defaults to dim ** -0.5.  A token that sees nothing,
    and a row of q outside starts, gets zeros; so do the rows of a sequence that
    starts gives more than most_new tokens or rows that q has not, which
    data_status() tells.  With return_lse also the f32 [tokens, q_heads] logarithm
    of the sum of exponentials (-inf where nothing is seen).  `workspace`: contiguous
    uint8 of at least `attention_workspace_bytes`, else allocated."""
    dt, dev, D = q.dtype, cache._dev, cache._dim
    if dt not in _HALF:
        raise RuntimeError("q must be bfloat16 or float16")
    T, H, qs = _heads("q", q, D, dt, dev)
    shape, st = table.shape, table.stride()
    if (len(shape) != 2 or table.dtype != torch.int32 or table.device != dev
            or not (st[1] == 1 or shape[1] <= 1 or table.is_contiguous())):
        raise RuntimeError("table must be int32 [seqs, max_pages], rows dense")
    B, P = shape
    lens_p = _index("lens", lens, B, torch.int32, dev)
    starts_p = None if starts is None else _index("starts", starts, B + 1, torch.int32, dev)
    with on_device(dev):
        out = torch.empty(T, H, D, dtype=dt, device=dev)
        lse = torch.empty(T, H, dtype=torch.float32, device=dev) if return_lse else None
        need = attention_workspace_bytes(cache._kv_heads, cache._page, D, H, P, B, T, most_new, window, dev)
        if workspace is not None:
            _req(workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.device == dev,
                 "workspace must be a contiguous uint8 tensor on the cache's device")
        elif need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        ws, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
        check(LIB.tans_b200_kv4_attention(
            cache._ref, q.data_ptr(), qs, H, table.data_ptr(), st[0], P, lens_p, starts_p, B, T, most_new,
            D ** -0.5 if scale is None else scale, window, out.data_ptr(), ptr(lse),
            ws, ws_bytes, _HALF[dt], _status(dev).data_ptr(), raw_stream(dev)))
    _post_check(dev)
    return (out, lse) if return_lse else out


__all__ = ["KV4Cache", "append", "read", "attention", "attention_workspace_bytes"]
