"""Residual + RMS norm, e4m3 quantisation and the e4m3 product with its
epilogue, against the formulas in 64 bits (GPU), and their refusals (CPU).

Bounds, elementwise.  u is half a unit in the last place of the output type
(2^-8 bf16, 2^-11 f16, 2^-24 f32).  A norm's f32 arithmetic adds under 2^-17
relative (a sum of at most 57344 squares in a tree of f32, a root, three
products).  An e4m3 value is within 2^-4 of its size, or 2^-10 of the scale
where it is subnormal.  A product of K terms accumulates in f32: at most K 2^-23
of the sum of the terms' sizes; activations have slope at most 1.13 and their
fast exponentials err by under 2^-17."""
from __future__ import annotations

import math

import pytest
import torch

from rans_vectoradd import fp8_linear
from rans_vectoradd._lib import LIB

HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}


def within(got, want, bound):
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), f"off by {float((d / bound.clamp_min(1e-300)).max())} of the bound"


def rand(shape, seed, dev, dtype=torch.float32, mul=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, device=dev, generator=g) * mul).to(dtype)


def e4m3(q):
    return q.view(torch.float8_e4m3fn).double()


def check_norm(x, w, r, eps=1e-6, quantize=False, **kw):
    s = x.double() + (r.double() if r is not None else 0)
    want = s / (s.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    u = HALF_ULP[x.dtype]
    # the f32 sum x + r rounds once before the norm
    slack = (2.0 ** -17 + 2.0 ** -20) * want.abs() + 2.0 ** -24 * (want / torch.where(s == 0, 1, s)).abs() * (
        x.double().abs() + (r.double().abs() if r is not None else 0))
    x0, r0 = x.clone(), None if r is None else r.clone()
    if quantize:
        q, scale, h = fp8_linear.add_rms_norm_e4m3(x, w, r, eps=eps, **kw)
        top = want.abs().amax(-1)
        within(scale, torch.where(top == 0, 1.0, top / 448), 2.0 ** -16 * top / 448 + 1e-30)
        within(e4m3(q) * scale.double()[:, None], want,
               (2.0 ** -4 + 2.0 ** -12) * want.abs() + 2.0 ** -10 * scale.double()[:, None] + slack)
    else:
        y, h = fp8_linear.add_rms_norm(x, w, r, eps=eps, **kw)
        within(y, want, 1.01 * u * want.abs() + TINY[x.dtype] + slack)
    if r0 is not None:
        assert torch.equal(h, (x0.float() + r0.float()).to(x.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 40), (2, 255), (5, 1024), (1, 5120), (7, 4099), (300, 5120),
                                       (2, 16384), (1, 32768), (2, 32776), (1, 57344), (1, 57341)])
def test_norm_matches_formula(cuda, dtype, rows, cols):
    x, r = rand((rows, cols), cols, cuda, dtype), rand((rows, cols), cols + 1, cuda, dtype, 3.0)
    w = (1 + rand((cols,), 2, cuda, mul=0.3)).to(dtype)
    for res in (r, None):
        for quantize in (False, True):
            check_norm(x, w, res, quantize=quantize)
    check_norm(x, w.float(), r, quantize=True)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [256, 250])
def test_norm_strided_rows_and_in_place(cuda, cols):
    base = rand((9, 3 * cols), 1, cuda, torch.bfloat16)
    x, r = base[:, cols:2 * cols], base[:, 2 * cols:]
    w = rand((cols,), 3, cuda, torch.bfloat16)
    check_norm(x, w, r)
    check_norm(x, w, r, quantize=True)
    want = (x.float() + r.float()).to(torch.bfloat16)
    keep = base[:, :cols].clone()
    _, h = fp8_linear.add_rms_norm(x, w, r, residual_out=r)
    assert h is r and torch.equal(r, want) and torch.equal(base[:, :cols], keep)
    x2, want2 = x.clone(), (x.float() + r.float()).to(torch.bfloat16)
    fp8_linear.add_rms_norm_e4m3(x2, w, r, residual_out=x2)
    assert torch.equal(x2, want2)
    # rows that start off 16 bytes
    odd = rand((5, cols + 1), 4, cuda, torch.float16)[:, 1:]
    check_norm(odd, w.half(), None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [1, 7, 9, 250, 1023, 4099, 32759, 32761])
def test_norm_rows_at_any_address(cuda, dtype, cols):
    """x, residual and the sum's rows begin the same or different distances past 16-byte boundaries, between NaN
    that must neither be read nor written over."""
    w = (1 + rand((cols,), 5, cuda, mul=0.3)).to(dtype)
    for seed, (at_x, at_r, at_h, gap) in enumerate([(0, 0, 0, 9), (1, 1, 1, 16), (1, 2, 1, 16), (3, 3, 5, 17), (8, 0, 8, 8)]):
        width = (cols + 15) // 8 * 8 + gap
        held = [torch.full((5, width), float("nan"), device=cuda, dtype=dtype) for _ in range(3)]
        x, r, h = (t[:, a:a + cols] for t, a in zip(held, (at_x, at_r, at_h)))
        x.copy_(rand((5, cols), seed, cuda, dtype))
        r.copy_(rand((5, cols), seed + 50, cuda, dtype, 2.0))
        for quantize in (False, True):
            check_norm(x, w, r, quantize=quantize, residual_out=h)
            check_norm(x, w.float(), None, quantize=quantize)
        for t in held:
            assert int(torch.isnan(t).sum()) == 5 * (width - cols)


@pytest.mark.gpu
def test_norm_zero_nan_inf_rows_and_empty(cuda):
    x = rand((5, 512), 0, cuda, torch.bfloat16)
    x[1] = 0
    x[2, 100] = float("nan")
    x[3, 7] = float("inf")
    w = torch.ones(512, dtype=torch.bfloat16, device=cuda)
    q, scale, h = fp8_linear.add_rms_norm_e4m3(x, w)
    assert h is x
    assert scale[1] == 1 and not q[1].any()
    assert torch.isnan(scale[2]) and torch.isnan(e4m3(q[2])).all()
    assert torch.isnan(scale[3])  # inf * 0
    q2, s2 = fp8_linear.quantize_tokens(x)
    assert s2[1] == 1 and not q2[1].any() and torch.isnan(s2[2]) and torch.isinf(s2[3])
    y, _ = fp8_linear.add_rms_norm(x, w)
    assert torch.isnan(y[2]).all() and not y[1].any()
    good = torch.tensor([0, 4], device=cuda)
    a, b, _ = fp8_linear.add_rms_norm_e4m3(x[good], w)
    assert torch.equal(q[good], a) and torch.equal(scale[good], b)
    none = x[:0]
    assert fp8_linear.add_rms_norm(none, w)[0].shape == (0, 512)
    assert fp8_linear.quantize_tokens(none)[1].shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 17408), (6, 777), (130, 64)])
def test_quantize_tokens(cuda, dtype, rows, cols):
    x = rand((rows, cols), 5, cuda, dtype)
    q, scale = fp8_linear.quantize_tokens(x)
    want = x.double()
    within(scale, want.abs().amax(-1) / 448, 2.0 ** -22 * want.abs().amax(-1) / 448)
    within(e4m3(q) * scale.double()[:, None], want,
           (2.0 ** -4 + 2.0 ** -12) * want.abs() + 2.0 ** -10 * scale.double()[:, None])


# ------------------------------------------------------------------- linear

def quantized(rows, cols, seed, dev, mul=1.0):
    x = rand((rows, cols), seed, dev, mul=mul)
    s = x.abs().amax(-1).clamp_min(1e-20) / 448
    return (x / s[:, None]).to(torch.float8_e4m3fn).view(torch.uint8), s


ACTS = {"none": lambda t: t, "relu": lambda t: t.clamp_min(0), "silu": lambda t: t * torch.sigmoid(t),
        "gelu_tanh": lambda t: 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))}


def check_linear(x8, xs, w8, ws, bias=None, act="none", mul=None, residual=None, dtype=torch.bfloat16, out=None):
    K = x8.shape[1]
    sc = xs.double()[:, None] * ws.double()
    pre = (e4m3(x8) @ e4m3(w8).t()) * sc
    size = (e4m3(x8).abs() @ e4m3(w8).abs().t()) * sc
    if bias is not None:
        pre, size = pre + bias.double(), size + bias.double().abs()
    want = ACTS[act](pre)
    bound = 1.13 * (K + 8) * 2.0 ** -23 * size + 2.0 ** -17 * want.abs()
    if mul is not None:
        want, bound = want * mul.double(), bound * mul.double().abs()
    if residual is not None:
        want = want + residual.double()
    got = fp8_linear.linear(x8, xs, w8, ws, bias=bias, act=act, mul=mul, residual=residual, dtype=dtype, out=out)
    within(got, want, bound + 1.01 * HALF_ULP[dtype] * want.abs() + TINY[dtype])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 128, 128), (1, 5120, 1024), (2, 129, 144), (15, 77, 4096),
                                   (17, 640, 5120), (33, 1000, 272), (64, 5120, 17408), (65, 256, 128),
                                   (129, 384, 1040), (200, 130, 2064), (257, 1024, 512), (512, 2048, 512),
                                   (700, 1111, 784), (1025, 300, 2048), (300, 6500, 272), (129, 12700, 144),
                                   (2000, 1700, 512), (1500, 5001, 400), (4100, 2600, 16), (384, 10240, 1024)])
def test_linear_matches_formula(cuda, m, n, k):
    x8, xs = quantized(m, k, m + n, cuda)
    w8, ws = quantized(n, k, k, cuda, 0.02)
    check_linear(x8, xs, w8, ws)
    b, mu, r = (rand(s, i, cuda, torch.bfloat16) for i, s in enumerate([(n,), (m, n), (m, n)]))
    check_linear(x8, xs, w8, ws, b, "silu", mu, r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m", [3, 300])
def test_linear_epilogues(cuda, dtype, act, m):
    n, k = 328, 256
    x8, xs = quantized(m, k, 1, cuda, 3.0)
    w8, ws = quantized(n, k, 2, cuda)
    b, mu, r = (rand(s, i, cuda, dtype) for i, s in enumerate([(n,), (m, n), (m, n)]))
    for has in range(8):
        check_linear(x8, xs, w8, ws, b if has & 1 else None, act, mu if has & 2 else None, r if has & 4 else None, dtype)
    want = fp8_linear.linear(x8, xs, w8, ws, residual=r, dtype=dtype)
    into = r.clone()
    assert fp8_linear.linear(x8, xs, w8, ws, residual=into, dtype=dtype, out=into) is into
    assert torch.equal(into, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 7, 32), (5, 333, 2064), (37, 130, 4096), (150, 335, 512), (131, 9601, 64), (260, 9600, 64),
                                   (513, 5003, 144)])
@pytest.mark.parametrize("into", ["mul", "residual", "none"])
def test_linear_at_any_address(cuda, m, n, k, into):
    """Rows of any count, operands and output two bytes past an alignment of 16, the output in an operand's place;
    nothing beyond its ends is written."""
    x8, xs = quantized(m, k, m, cuda)
    w8, ws = quantized(n, k, n, cuda, 0.1)
    held = {name: torch.full((m * n + 20,), 77.0, dtype=torch.bfloat16, device=cuda) for name in ("mul", "residual", "none")}
    at = {name: t[1:1 + m * n].view(m, n) for name, t in held.items()}
    at["mul"].copy_(rand((m, n), 1, cuda))
    at["residual"].copy_(rand((m, n), 2, cuda))
    b, mul, residual = rand((n,), 3, cuda, torch.bfloat16), at["mul"].clone(), at["residual"].clone()
    want = check_linear(x8, xs, w8, ws, b, "silu", mul, residual)
    got = fp8_linear.linear(x8, xs, w8, ws, bias=b, act="silu", mul=at["mul"], residual=at["residual"], out=at[into])
    assert got is at[into] and torch.equal(got, want)
    for t in held.values():
        assert t[0] == 77 and bool((t[1 + m * n:] == 77).all())


@pytest.mark.gpu
def test_linear_is_deterministic_and_takes_an_empty_batch(cuda):
    x8, xs = quantized(48, 17408, 3, cuda)
    w8, ws = quantized(640, 17408, 4, cuda)
    a = fp8_linear.linear(x8, xs, w8, ws)
    assert all(torch.equal(a, fp8_linear.linear(x8, xs, w8, ws)) for _ in range(4))
    assert fp8_linear.linear(x8[:0], xs[:0], w8, ws).shape == (0, 640)


@pytest.mark.gpu
def test_linear_nan_stays_in_its_row_and_token(cuda):
    x8, xs = quantized(20, 512, 3, cuda)
    w8, ws = quantized(130, 512, 4, cuda)
    x8[7, 3] = 0x7F
    w8[100, 5] = 0xFF
    y = fp8_linear.linear(x8, xs, w8, ws)
    bad = torch.zeros(20, 130, dtype=torch.bool, device=cuda)
    bad[7] = True
    bad[:, 100] = True
    assert torch.equal(torch.isnan(y), bad)


@pytest.mark.gpu
def test_a_chain_on_a_side_stream(cuda):
    """Norm, product, quantisation and product back to back on a stream of their own, each
    reading what the one before has just written, equal to the same calls one by one."""
    h, w = rand((40, 512), 1, cuda, torch.bfloat16), torch.ones(512, dtype=torch.bfloat16, device=cuda)
    up, us = quantized(1024, 512, 2, cuda, 0.05)
    down, ds = quantized(512, 1024, 3, cuda, 0.05)
    x = rand((40, 512), 5, cuda, torch.bfloat16)

    def step(sync):
        r, y = h, x
        for _ in range(4):
            q, s, r = fp8_linear.add_rms_norm_e4m3(y, w, r)
            sync()
            a = fp8_linear.linear(q, s, up, us, act="gelu_tanh")
            sync()
            q, s = fp8_linear.quantize_tokens(a)
            sync()
            y = fp8_linear.linear(q, s, down, ds)
            sync()
        return r, y

    want = step(torch.cuda.synchronize)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(lambda: None)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ----------------------------------------------------------------- refusals

def test_python_refusals():
    x = torch.zeros(2, 32)
    for call in (lambda: fp8_linear.add_rms_norm(x, torch.zeros(32)), lambda: fp8_linear.quantize_tokens(x),
                 lambda: fp8_linear.linear(x.to(torch.uint8), torch.zeros(2), x.to(torch.uint8), torch.zeros(2))):
        with pytest.raises(RuntimeError):
            call()


def test_c_refusals():
    """Argument errors come back as a status and a message, before any launch."""
    p = 256  # an aligned address that is never followed
    err = lambda: LIB.tans_b200_last_error().decode()  # noqa: E731
    norm = lambda rows=1, cols=8, y=p, q=None, s=None, res=None, h=None, eps=1e-6, wt=0, dt=0: (  # noqa: E731
        LIB.tans_b200_add_rms_norm(p, 8, res, 8, p, wt, eps, h, 8, y, q, s, rows, cols, dt, None))
    for kw, word in (({"rows": -1}, "rows"), ({"cols": 0}, "cols"), ({"cols": 57345}, "cols"), ({"y": None}, "needed"),
                     ({"q": p}, "needed"), ({"res": p}, "needed"), ({"eps": -1.0}, "eps"), ({"wt": 1}, "weight"),
                     ({"dt": 3, "wt": 3}, "type"), ({"eps": float("nan")}, "eps")):
        assert norm(**kw) == 1 and word in err(), (kw, err())
    assert norm(rows=0) == 0
    lin = lambda x=p, w=p, m=1, n=8, k=16, act=0, dt=0: LIB.tans_b200_linear(  # noqa: E731
        x, p, w, p, None, act, None, None, p, m, n, k, dt, None, None)
    for kw, word in (({"k": 15}, "multiple"), ({"k": 0}, "multiple"), ({"n": 0}, "rows"), ({"act": 4}, "activation"),
                     ({"x": 8}, "aligned"), ({"w": None}, "needed"), ({"m": -1}, "rows")):
        assert lin(**kw) == 1 and word in err(), (kw, err())
    assert lin(m=0) == 0
    assert LIB.tans_b200_quantize_tokens(None, 8, p, p, 1, 8, 0, None) == 1


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    x = torch.zeros(2, 32, dtype=torch.bfloat16, device=cuda)
    w = torch.zeros(32, dtype=torch.bfloat16, device=cuda)
    x8 = torch.zeros(2, 32, dtype=torch.uint8, device=cuda)
    s = torch.ones(2, device=cuda)
    for call in (lambda: fp8_linear.add_rms_norm(x, w[:31]), lambda: fp8_linear.add_rms_norm(x.t(), w[:2]),
                 lambda: fp8_linear.add_rms_norm(x, w, x.half()), lambda: fp8_linear.add_rms_norm(x, w.half()),
                 lambda: fp8_linear.add_rms_norm(x, w, residual_out=x), lambda: fp8_linear.add_rms_norm(x.double(), w),
                 lambda: fp8_linear.linear(x8, s, x8[:, :16], s), lambda: fp8_linear.linear(x8, s, x8, s.double()),
                 lambda: fp8_linear.linear(x8, s, x8, s, act="tanh"), lambda: fp8_linear.linear(x8, s[:1], x8, s),
                 lambda: fp8_linear.linear(x8, s, x8, s, bias=w), lambda: fp8_linear.linear(x8, s, x8, s, dtype=torch.float32),
                 lambda: fp8_linear.linear(x8, s, x8, s, residual=x[:, :2]),
                 lambda: fp8_linear.linear(x8[:, :24].contiguous(), s, x8[:, :24].contiguous(), s)):
        with pytest.raises(RuntimeError):
            call()
