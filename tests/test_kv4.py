"""The paged 4-bit cache: append with rotation, read, attention (GPU, against
the definitions), and refusals (CPU).

What `append` stores is defined bit by bit (f32 products and sums rounded one
by one, round to nearest even), so codes and scales are compared for equality
with an implementation in elementary torch operations on the CPU.

Attention's bounds, elementwise, with A = sum of p|v| over the keys: u|o| for
the output's rounding (u = 2^-8 bf16, 2^-11 f16); weights p enter the second
product in f16 (2^-11 A, and 2^-25 a key below f16's normal range, in units of
the largest value); a score of D f32-accumulated products errs by at most
e = scale (D + 16) 2^-23 sum|q||k| + 2^-20 of its size, which moves p by e."""
from __future__ import annotations

import math

import pytest
import torch

from rans_vectoradd import _C, kv4
from rans_vectoradd._lib import LIB, KV4

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def gen(seed, dev="cpu"):
    return torch.Generator(device=dev).manual_seed(seed)


def to_codes(x):
    """Reference quantisation of f32 [..., D] on the CPU: packed codes, e4m3 scale bytes."""
    b = x.unflatten(-1, (-1, 16))
    s8 = (b.abs().amax(-1) / torch.tensor(6.0)).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = s8.float()[..., None]
    r = torch.where(s == 0, torch.zeros_like(b), b / torch.where(s == 0, torch.ones_like(s), s))
    a = r.abs().double()[..., None]
    # nearest code, the even one of two equally near
    d = (a - E2M1.double()).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    even = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0], dtype=torch.bool)
    pick = torch.where((near & even).any(-1, keepdim=True), near & even, near)
    code = pick.int().argmax(-1) + 8 * (torch.signbit(r)).int()
    code = code.flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), s8.view(torch.uint8)


def from_codes(codes, scales):
    """f64 values [..., D]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = E2M1.double().to(codes.device)[c & 7] * torch.where(c > 7, -1.0, 1.0)
    return (v.unflatten(-1, (-1, 16)) * scales.view(torch.float8_e4m3fn).double()[..., None]).flatten(-2)


def rotate32(x, cos, sin, interleaved):
    """f32 on the CPU; x [T, H, D]."""
    n = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    out = x.clone()
    i = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., i[0]], x[..., i[1]]
    out[..., i[0]] = a * c - b * s
    out[..., i[1]] = b * c + a * s
    return out


def angles(top, n, base=10000.0):
    a = torch.arange(top, dtype=torch.float64)[:, None] * base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
    return a.cos().float(), a.sin().float()


# ------------------------------------------------------------ append and read

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,q_heads,dim,page,half,interleaved", [
    (1, 1, 1, 64, 1, 32, False), (7, 2, 6, 128, 16, 64, False), (33, 8, 8, 128, 8, 64, True), (5, 1, 9, 256, 4, 128, False),
    (64, 4, 4, 64, 32, 16, False), (9, 3, 3, 128, 2, 7, False), (9, 3, 3, 128, 64, 13, True), (20, 2, 4, 256, 16, 32, True),
    (130, 5, 5, 128, 16, 0, False)])
def test_append_and_read(cuda, dtype, tokens, heads, q_heads, dim, page, half, interleaved):
    g = gen(tokens + dim)
    pages = -(-tokens // page) + 2
    k, v = torch.randn(tokens, heads, dim, generator=g).to(dtype), (3 * torch.randn(tokens, heads, dim, generator=g)).to(dtype)
    q = torch.randn(tokens, q_heads, dim, generator=g).to(dtype)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    pos = torch.randint(0, 500, (tokens,), generator=g)
    cos, sin = angles(500, half)
    cache = kv4.KV4Cache.allocate(pages, heads, page, dim, cuda)
    junk = torch.randint(0, 256, cache.k_codes.shape, generator=g, dtype=torch.uint8)
    cache.k_codes.copy_(junk)
    rot = dict(positions=pos.to(cuda), cos=cos.to(cuda), sin=sin.to(cuda)) if half else {}
    got_q = kv4.append(cache, k.to(cuda), v.to(cuda), slots.to(cuda), q=q.to(cuda), interleaved=interleaved, **rot)
    turn = (lambda x: rotate32(x.float(), cos[pos], sin[pos], interleaved)) if half else (lambda x: x.float())
    assert torch.equal(got_q.cpu(), turn(q).to(dtype))
    at = (slots // page, slots % page)
    for name, x in (("k", turn(k)), ("v", v.float())):
        codes, scales = to_codes(x)
        held_c, held_s = getattr(cache, name + "_codes").cpu(), getattr(cache, name + "_scales").cpu()
        assert torch.equal(held_s[at[0], :, at[1]], scales)
        assert torch.equal(from_codes(held_c, held_s)[at[0], :, at[1]], from_codes(codes, scales))
        nz = held_c[at[0], :, at[1]] != codes  # codes may differ in the sign of a zero alone
        assert not nz.any() or torch.equal(from_codes(held_c[at[0], :, at[1]], scales), from_codes(codes, scales))
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(cache.k_codes.cpu().transpose(1, 2)[rest], junk.transpose(1, 2)[rest])
    assert not cache.v_codes.cpu().transpose(1, 2)[rest].any()
    for out_t in (torch.bfloat16, torch.float16, torch.float32):
        rk, rv = kv4.read(cache, slots.to(cuda), out_t)
        for name, r in (("k", rk), ("v", rv)):
            want = from_codes(getattr(cache, name + "_codes"), getattr(cache, name + "_scales"))
            assert torch.equal(r.double(), want[at[0].to(cuda), :, at[1].to(cuda)])
    assert _C.data_status() == 0


@pytest.mark.gpu
def test_append_rounding_edges(cuda):
    """Ties of codes and scales, values past the largest scale, zeros, blocks with NaN and inf."""
    x = torch.zeros(1, 1, 128)
    x[0, 0, :16] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6])
    x[0, 0, 16] = 6.375           # scale 1.0625, half way between 1 and 1.125
    x[0, 0, 32] = 2.0 ** -8 * 6   # a subnormal scale
    x[0, 0, 48] = 2.0 ** -12      # scale rounds to 0
    x[0, 0, 64:66] = torch.tensor([30000.0, -5000.0])
    x[0, 0, 80], x[0, 0, 96] = float("inf"), float("nan")
    x = x.to(torch.bfloat16)
    cache = kv4.KV4Cache.allocate(1, 1, 1, 128, cuda)
    slot = torch.zeros(1, dtype=torch.int64, device=cuda)
    kv4.append(cache, x.to(cuda), x.to(cuda), slot)
    k, v = kv4.read(cache, slot, torch.float32)
    k = k.cpu()[0, 0]
    assert torch.equal(k, v.cpu()[0, 0]) or torch.isnan(k).any()
    assert k[:16].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, -6]
    assert k[16] == 6.0 and k[32] == 2.0 ** -8 * 6 and not k[48:64].any()
    assert k[64] == 448 * 6 and k[65] == -448 * 6
    assert k[80] == 448 * 6 and not k[81:96].any()
    assert torch.isnan(k[96:112]).all() and not k[112:].any()


@pytest.mark.gpu
def test_append_gains_strides_skips(cuda):
    g = gen(3)
    T, H, D = 12, 2, 128
    gains = [torch.tensor([0.01, 7.0]), torch.tensor([300.0, 0.5])]
    cache = kv4.KV4Cache.allocate(3, H, 8, D, cuda, *(x.to(cuda) for x in gains))
    qkv = (torch.randn(T, 8 * D, generator=g) * 0.01).to(torch.bfloat16)
    q, k, v = qkv[:, :4 * D].view(T, 4, D), qkv[:, 4 * D:6 * D].view(T, H, D), qkv[:, 6 * D:].view(T, H, D)
    dq = qkv.to(cuda)
    slots = torch.randperm(24, generator=g)[:T]
    slots[3] = -1
    cos, sin = angles(64, 64)
    pos = torch.arange(T) * 5
    out = kv4.append(cache, dq[:, 4 * D:6 * D].view(T, H, D), dq[:, 6 * D:].view(T, H, D), slots.to(cuda),
                     positions=pos.to(cuda), cos=cos.to(cuda), sin=sin.to(cuda), q=dq[:, :4 * D].view(T, 4, D))
    assert torch.equal(out.cpu(), rotate32(q.float(), cos[pos], sin[pos], False).to(torch.bfloat16))
    keep = slots >= 0
    rk, rv = (t.cpu() for t in kv4.read(cache, slots.to(cuda), torch.float32))
    assert not rk[3].any() and not rv[3].any()
    for got, x, gain in ((rk, rotate32(k.float(), cos[pos], sin[pos], False), gains[0]), (rv, v.float(), gains[1])):
        codes, scales = to_codes(x / gain[:, None])
        want = from_codes(codes, scales) * gain.double()[:, None]
        assert torch.allclose(got.double()[keep], want[keep], rtol=2.0 ** -22, atol=0)
    assert _C.data_status() == 0


@pytest.mark.gpu
def test_append_flags_bad_indices(cuda):
    T, H, D = 4, 1, 64
    cache = kv4.KV4Cache.allocate(2, H, 4, D, cuda)
    x = torch.ones(T, H, D, dtype=torch.float16, device=cuda)
    slots = torch.tensor([0, 8, 1 << 40, 3], device=cuda)
    _C.data_status()
    kv4.append(cache, x, x, slots)
    assert _C.data_status() == 16
    held = kv4.read(cache, torch.arange(8, device=cuda))[0]
    assert held[0].all() and held[3].all() and not held[[1, 2, 4, 5, 6, 7]].any()
    cos, sin = (t.to(cuda) for t in angles(10, 8))
    ok = torch.arange(4, device=cuda)
    q = kv4.append(cache, x, x, ok, positions=torch.tensor([0, 10, -1, 9], device=cuda), cos=cos, sin=sin, q=x)
    assert _C.data_status() == 16
    assert torch.equal(q[1:3], x[1:3]) and not torch.equal(q[3], x[3])
    kv4.read(cache, torch.tensor([8], device=cuda))
    assert _C.data_status() == 16
    assert kv4.append(cache, x[:0], x[:0], ok[:0], q=x[:0]).shape == (0, H, D)


# ------------------------------------------------------------------ attention

def build(lens, news, heads, group, dim, page, dtype, seed, dev, spread=1.0, gains=False):
    """A cache of random tokens in shuffled pages, queries, and the f64 keys and values."""
    g = gen(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 3
    shape = (pages, heads, page)
    cache = {}
    for n in "kv":
        codes, scales = to_codes(torch.randn(*shape, dim, generator=g) * (spread if n == "k" else 1.0))
        cache[n + "_codes"], cache[n + "_scales"] = codes, scales
    if gains:
        cache["k_gain"], cache["v_gain"] = torch.rand(heads, generator=g) + 0.5, torch.rand(heads, generator=g) * 3
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max(counts + [1]) + 1), -1, dtype=torch.int32)
    at, keys, vals = 0, [], []
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
        idx = table[b, :c].long()
        for n, to in (("k", keys), ("v", vals)):
            x = from_codes(cache[n + "_codes"][idx], cache[n + "_scales"][idx]).transpose(0, 1).flatten(1, 2)[:, :lens[b]]
            to.append(x * (cache[n + "_gain"].double()[:, None, None] if gains else 1))
    q = torch.randn(sum(news), heads * group, dim, generator=g).to(dtype)
    starts = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32)
    dc = kv4.KV4Cache(**{n: t.to(dev) for n, t in cache.items()})
    return dc, q, table, torch.tensor(lens, dtype=torch.int32), starts, keys, vals


def reference(q, keys, vals, lens, news, group, scale, window):
    """(out, lse, bound of out, bound of lse) in f64."""
    outs, lses, bo, bl = [], [], [], []
    u = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    at, D = 0, q.shape[2]
    for b, n in enumerate(news):
        x = q[at:at + n].double()
        at += n
        k, v = keys[b].repeat_interleave(group, 0), vals[b].repeat_interleave(group, 0)
        s = torch.einsum("thd,hld->thl", x, k) * scale
        size = torch.einsum("thd,hld->thl", x.abs(), k.abs()) * abs(scale)
        last = lens[b] - n + torch.arange(n)[:, None]
        key = torch.arange(lens[b])[None]
        seen = (key <= last) & ((key > last - window) if window else (key >= 0))
        s = torch.where(seen[:, None], s, -math.inf)
        top = s.amax(-1, keepdim=True) if lens[b] else torch.full((n, x.shape[1], 1), -math.inf, dtype=torch.float64)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp(s - top)
        tot = p.sum(-1, keepdim=True)
        w = torch.where(tot > 0, p / tot, 0.0)
        o = torch.einsum("thl,hld->thd", w, v)
        a = torch.einsum("thl,hld->thd", w, v.abs())
        fin = torch.where(seen[:, None], s.abs(), 0.0)
        e = ((D + 16) * 2.0 ** -23 * size + 2.0 ** -20 * fin + 2.0 ** -20)
        e = torch.where(seen[:, None], e, 0.0).amax(-1, keepdim=True) if lens[b] else torch.zeros_like(tot)
        outs.append(o)
        big = v.abs().amax() if v.numel() else torch.tensor(0.0)
        bo.append(1.01 * u * o.abs() + (2.0 ** -11 + 2 * e + 2.0 ** -18) * a + lens[b] * 2.0 ** -25 * big + 2.0 ** -25)
        lse = torch.log(tot) + top
        lses.append(lse[..., 0])
        bl.append((e + 2.0 ** -18 + 2.0 ** -21 * torch.where(tot > 0, lse.abs(), 0.0))[..., 0])
    return torch.cat(outs), torch.cat(lses), torch.cat(bo), torch.cat(bl)


def check_attention(cuda, lens, news, heads, group, dim, page, dtype, window=0, seed=0, scale=None, spread=1.0,
                    gains=False, use_starts=True):
    cache, q, table, ln, starts, keys, vals = build(lens, news, heads, group, dim, page, dtype, seed, cuda, spread, gains)
    sc = dim ** -0.5 if scale is None else scale
    want, lse, bo, bl = reference(q, keys, vals, lens, news, group, sc, window)
    kw = dict(starts=starts.to(cuda), most_new=max(news)) if use_starts else {}
    _C.data_status()
    got, got_lse = kv4.attention(cache, q.to(cuda), table.to(cuda), ln.to(cuda), scale=scale, window=window,
                                 return_lse=True, **kw)
    assert _C.data_status() == 0
    d = (got.cpu().double() - want).abs()
    assert bool((d <= bo).all()), f"out: {float((d / bo).max())} of the bound"
    fin = torch.isfinite(lse)
    assert torch.equal(torch.isneginf(got_lse.cpu()), torch.isneginf(lse))
    dl = (got_lse.cpu().double() - lse).abs()[fin]
    assert bool((dl <= bl[fin]).all()), f"lse: {float((dl / bl[fin]).max())} of the bound"
    again = kv4.attention(cache, q.to(cuda), table.to(cuda), ln.to(cuda), scale=scale, window=window, **kw)
    assert torch.equal(again, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,group,page", [(1, 1, 16), (2, 4, 32), (2, 7, 8), (1, 16, 64), (1, 33, 16), (3, 5, 1)])
def test_attention_one_new_token(cuda, dtype, dim, heads, group, page):
    lens = [1, 2, 15, 16, 17, 0, 63, 64, 65, 200, 129]
    check_attention(cuda, lens, [1] * len(lens), heads, group, dim, page, dtype, use_starts=False, seed=dim + group)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 100])
def test_attention_several_new_tokens_and_windows(cuda, dim, window):
    """Causal rows, rows that see nothing (fewer tokens held than new), sequences with no new token."""
    lens, news = [40, 3, 0, 130, 7, 65, 300], [5, 5, 2, 33, 0, 1, 17]
    check_attention(cuda, lens, news, 2, 3, dim, 16, torch.bfloat16, window=window, seed=window)
    check_attention(cuda, lens, news, 1, 8, dim, 4, torch.float16, window=window, seed=window + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,lens,heads,group,dtype", [
    (128, [5000, 1, 2500], 2, 4, torch.bfloat16), (64, [9001], 1, 8, torch.float16), (256, [4097, 4095], 1, 2, torch.bfloat16),
    (128, [30011], 1, 1, torch.bfloat16), (128, [700] * 40, 4, 2, torch.float16)])
def test_attention_long_sequences(cuda, dim, lens, heads, group, dtype):
    check_attention(cuda, lens, [1] * len(lens), heads, group, dim, 16, dtype, seed=len(lens))
    check_attention(cuda, lens, [2] * len(lens), heads, group, dim, 64, dtype, window=2000, seed=len(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("spread,scale", [(30.0, None), (1.0, 0.0), (4.0, -0.3), (1e-3, 5.0), (100.0, 1.0)])
def test_attention_scales_and_gains(cuda, spread, scale):
    """Peaked and flat weights, a scale of 0 and a negative one, per-head gains."""
    check_attention(cuda, [333, 1000], [1, 1], 2, 4, 128, 32, torch.bfloat16, spread=spread, scale=scale, gains=True,
                    use_starts=False, seed=5)


@pytest.mark.gpu
def test_attention_ignores_what_is_masked(cuda):
    """NaN scales in places past a sequence's end, before its window, and in a new token that an earlier one must
    not see; table entries past its pages."""
    lens, news, page = [37, 20], [3, 1], 16
    cache, q, table, ln, starts, keys, vals = build(lens, news, 1, 4, 128, page, torch.bfloat16, 9, cuda)
    args = lambda c: dict(starts=starts.to(cuda), most_new=3, return_lse=True)  # noqa: E731
    want, lse = kv4.attention(cache, q.to(cuda), table.to(cuda), ln.to(cuda), **args(cache))
    for name in "kv":
        for b, n in enumerate(lens):
            last = int(table[b, (n - 1) // page])
            getattr(cache, name + "_scales")[last, :, (n - 1) % page + 1:] = 0x7F
            getattr(cache, name + "_codes")[last, :, (n - 1) % page + 1:] = 0xFF
    wild = table.clone()
    wild[0, 3:], wild[1, 2:] = 1 << 30, -7
    got, got_lse = kv4.attention(cache, q.to(cuda), wild.to(cuda), ln.to(cuda), **args(cache))
    assert torch.equal(got, want) and torch.equal(got_lse, lse)
    # the last new token of sequence 0 turns NaN: only its own row may see it
    for name, see_lse in (("v", False), ("k", True)):
        keep = getattr(cache, name + "_scales").clone()
        getattr(cache, name + "_scales")[int(table[0, 2]), :, 36 % page, 2] = 0xFF
        got, got_lse = kv4.attention(cache, q.to(cuda), table.to(cuda), ln.to(cuda), **args(cache))
        assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])
        assert torch.isnan(got[2] if see_lse else got[2, :, 32:48]).all()
        assert torch.isnan(got_lse[2]).all() == see_lse
        if not see_lse:
            assert torch.equal(got[2, :, :32], want[2, :, :32]) and torch.equal(got[2, :, 48:], want[2, :, 48:])
        getattr(cache, name + "_scales").copy_(keep)
    # a window of 4: a NaN at key 32 is in nobody's sight, one at key 33 in that of the second-to-last tokens
    w = dict(window=3, **args(cache))
    want, _ = kv4.attention(cache, q.to(cuda), table.to(cuda), ln.to(cuda), **w)
    cache.v_scales[int(table[0, 2]), :, 0] = 0x7F     # key 32: token 0 sees 32..34
    got, _ = kv4.attention(cache, q.to(cuda), table.to(cuda), ln.to(cuda), **w)
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], want[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("page", [4, 32])
@pytest.mark.parametrize("columns", [20, 300])  # too few pages at most to split the keys, and enough
@pytest.mark.parametrize("before,after", [(0, 0), (0, 3), (2, 1)])
def test_attention_takes_views_and_spare_rows(cuda, page, columns, before, after):
    """q between other columns of one tensor, a table within a wider one, rows of q that no sequence has."""
    cache, q, table, ln, starts, keys, vals = build([70, 33, 9], [2, 1, 4], 2, 3, 128, page, torch.bfloat16, 3, cuda)
    want, lse, bo, bl = reference(q, keys, vals, ln.tolist(), [2, 1, 4], 3, 128 ** -0.5, 0)
    tokens = before + 7 + after
    wide = torch.full((tokens, 6 * 128 + 264), float("nan"), dtype=torch.bfloat16, device=cuda)
    view = wide[:, 264:].unflatten(1, (6, 128))
    view[before:before + 7] = q.to(cuda)
    tables = torch.full((3, columns + 5), 1 << 29, dtype=torch.int32, device=cuda)
    tables[:, 3:3 + table.shape[1]] = table.to(cuda)
    del wide
    torch.full((tokens, 6, 128), float("nan"), dtype=torch.bfloat16, device=cuda)  # what the output's memory may hold
    _C.data_status()
    got, got_lse = kv4.attention(cache, view, tables[:, 3:-2], ln.to(cuda), starts=starts.to(cuda) + before, most_new=4,
                                 return_lse=True)
    assert _C.data_status() == 0
    got, got_lse = got.cpu(), got_lse.cpu()
    own = slice(before, before + 7)
    assert bool(((got[own].double() - want).abs() <= bo).all()) and bool(((got_lse[own].double() - lse).abs() <= bl).all())
    spare = torch.ones(tokens, dtype=torch.bool)
    spare[own] = False
    assert not got[spare].any() and torch.isneginf(got_lse[spare]).all()
    none, none_lse = kv4.attention(cache, view, tables[:0], ln[:0].to(cuda), starts=starts[:1].to(cuda), return_lse=True)
    assert not none.any() and torch.isneginf(none_lse).all()


@pytest.mark.gpu
def test_attention_flags_bad_metadata(cuda):
    cache, q, table, ln, starts, *_ = build([40, 40], [1, 1], 1, 2, 64, 16, torch.bfloat16, 1, cuda)
    run = lambda t=table, n=ln, **kw: kv4.attention(cache, q.to(cuda), t.to(cuda), n.to(cuda), **kw)  # noqa: E731
    _C.data_status()
    want = run()
    assert _C.data_status() == 0
    for bad in (-1, cache.k_codes.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 1] = bad
        got = run(t)
        assert _C.data_status() == 16 and torch.equal(got[1], want[1])
    for bad in (-5, 65, 2 ** 31 - 1):
        got = run(n=torch.tensor([bad, 40], dtype=torch.int32))
        assert _C.data_status() == 16 and torch.equal(got[1], want[1])
    for bad in ([0, 2, 2], [0, 0, 3], [-1, 1, 2], [0, 2 ** 31 - 1, 2]):
        run(starts=torch.tensor(bad, dtype=torch.int32, device=cuda))
        assert _C.data_status() == 16


@pytest.mark.gpu
def test_attention_offsets_past_32_bits(cuda):
    """A cache whose code arrays pass 2^31 bytes: the sequence lies in its last pages."""
    pages, heads, page, dim = (1 << 31) // (8 * 128 * 64) + 40, 8, 128, 128
    small, q, table, ln, starts, keys, vals = build([300], [1], heads, 2, dim, page, torch.bfloat16, 2, cuda)
    want = kv4.attention(small, q.to(cuda), table.to(cuda), ln.to(cuda))
    arrays = {}
    n = small.k_codes.shape[0]
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        src = getattr(small, name)
        big = torch.empty((pages, *src.shape[1:]), dtype=torch.uint8, device=cuda)
        big[-n:] = src
        arrays[name] = big
    cache = kv4.KV4Cache(**arrays)
    t = torch.where(table >= 0, table + (pages - n), table)
    assert arrays["k_codes"].numel() > 2 ** 31
    assert torch.equal(kv4.attention(cache, q.to(cuda), t.to(cuda), ln.to(cuda)), want)
    slot = torch.tensor([pages * page - 1], device=cuda)
    x = torch.randn(1, heads, dim, device=cuda).to(torch.bfloat16)
    kv4.append(cache, x, x, slot)
    k, v = kv4.read(cache, slot)
    assert torch.equal(k, v) and k.any()


@pytest.mark.gpu
def test_step_on_a_side_stream_and_in_a_graph(cuda):
    """append then attention on a stream of their own, and replayed from a CUDA graph."""
    heads, group, dim, page = 2, 4, 128, 16
    cache, q, table, ln, starts, *_ = build([50, 200], [1, 1], heads, group, dim, page, torch.bfloat16, 4, cuda)
    k = torch.randn(2, heads, dim, generator=gen(1)).to(torch.bfloat16).to(cuda)
    slots = (table[torch.arange(2), (ln - 1) // page].long() * page + (ln - 1) % page).to(cuda)
    t, n, q = table.to(cuda), ln.to(cuda), q.to(cuda)

    def step():
        qq = kv4.append(cache, k, k, slots, q=q)
        return kv4.attention(cache, qq, t, n)

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    cache.k_codes.view(-1)[:] = cache.k_codes.view(-1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------------------ refusals

def test_c_refusals():
    p = 256  # an aligned address that is never followed
    err = lambda: LIB.tans_b200_last_error().decode()  # noqa: E731

    def cache(**kw):
        f = dict(k_codes=p, k_scales=p, v_codes=p, v_scales=p, k_gain=None, v_gain=None, pages=4, heads=2, page_size=16, dim=128)
        f.update(kw)
        return KV4(*f.values())

    def append(c, k=p, ks=256, q=None, qo=None, half=0, pos=None, tokens=1, dt=0):
        import ctypes
        return LIB.tans_b200_kv4_append(ctypes.byref(c), k, ks, p, 256, p, q, 256, 2, qo, pos, pos, pos, 10, half, 0,
                                        tokens, dt, None, None)

    for kw, word in (({"k_codes": None}, "null"), ({"pages": 0}, "positive"), ({"page_size": 24}, "power of two"),
                     ({"page_size": 1 << 17}, "power of two"), ({"dim": 96}, "64, 128 or 256"), ({"v_scales": 8}, "aligned"),
                     ({"heads": 0}, "positive")):
        assert append(cache(**kw)) == 1 and word in err(), (kw, err())
    for kw, word in (({"k": None}, "needed"), ({"k": 8}, "aligned"), ({"ks": 129}, "multiples"), ({"q": p}, "needed"),
                     ({"q": p, "qo": p}, "must not be q"), ({"half": 65}, "half"), ({"half": 8}, "half"), ({"tokens": -1}, "tokens"),
                     ({"dt": 2}, "type")):
        assert append(cache(), **kw) == 1 and word in err(), (kw, err())
    assert append(cache(), tokens=0) == 0

    def attend(c=None, H=4, seqs=1, tokens=1, most=1, window=0, q=p, starts=None, pages=4):
        import ctypes
        return LIB.tans_b200_kv4_attention(ctypes.byref(c or cache()), q, 512, H, p, 4, pages, p, starts, seqs, tokens,
                                           most, 1.0, window, p, None, None, 0, 0, None, None)

    for kw, word in (({"H": 3}, "multiple"), ({"H": 0}, "multiple"), ({"most": 0}, "most_new"), ({"window": -1}, "window"),
                     ({"tokens": 2}, "starts"), ({"q": None}, "needed"), ({"q": 8}, "aligned"), ({"pages": 1 << 30}, "holds at most"),
                     ({"seqs": 65536, "tokens": 65536}, "seqs")):
        assert attend(**kw) == 1 and word in err(), (kw, err())
    assert attend(seqs=0, tokens=0) == 0


def test_python_refusals():
    with pytest.raises(RuntimeError, match="contiguous CUDA"):
        kv4.KV4Cache.allocate(2, 2, 16, 128, device="cpu")
    with pytest.raises(RuntimeError, match="power of two"):
        kv4.KV4Cache.allocate(2, 2, 24, 128, device="cpu")
    with pytest.raises(RuntimeError, match="dim 64"):
        kv4.KV4Cache.allocate(2, 2, 16, 96, device="cpu")


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    cache = kv4.KV4Cache.allocate(4, 2, 16, 128, cuda)
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device=cuda)
    s = torch.arange(3, device=cuda)
    cos, sin = (t.to(cuda) for t in angles(8, 64))
    wide = torch.zeros(8, 65, device=cuda)
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16, device=cuda)
    table, lens = torch.zeros(3, 2, dtype=torch.int32, device=cuda), torch.ones(3, dtype=torch.int32, device=cuda)
    for call in (lambda: kv4.append(cache, x, x.half(), s), lambda: kv4.append(cache, x[:, :1], x[:, :1], s),
                 lambda: kv4.append(cache, x, x, s.int()), lambda: kv4.append(cache, x, x, s[:2]),
                 lambda: kv4.append(cache, x, x, s, positions=s), lambda: kv4.append(cache, x, x, s, cos=cos, sin=sin),
                 lambda: kv4.append(cache, x, x, s, positions=s, cos=wide, sin=wide),
                 lambda: kv4.append(cache, x.transpose(0, 1), x, s), lambda: kv4.append(cache, x, x, s, q=q[:2]),
                 lambda: kv4.append(cache, x.float(), x.float(), s), lambda: kv4.append(cache, x[..., ::2], x[..., ::2], s),
                 lambda: kv4.read(cache, s.int()), lambda: kv4.read(cache, s, torch.float64),
                 lambda: kv4.attention(cache, q[:, :3], table, lens), lambda: kv4.attention(cache, q, table.long(), lens),
                 lambda: kv4.attention(cache, q, table[:2], lens), lambda: kv4.attention(cache, q.float(), table, lens),
                 lambda: kv4.attention(cache, q, table, lens[:2]), lambda: kv4.attention(cache, q, table, lens, most_new=0),
                 lambda: kv4.attention(cache, q, table, lens, starts=lens), lambda: kv4.attention(cache, q, table, lens, window=-1),
                 lambda: kv4.KV4Cache(cache.k_codes, cache.k_codes, cache.v_codes, cache.v_scales),
                 lambda: kv4.KV4Cache(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, k_gain=cos[0])):
        with pytest.raises(RuntimeError):
            call()
