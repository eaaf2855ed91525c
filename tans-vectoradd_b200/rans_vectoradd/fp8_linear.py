"""e4m3 activations and the e4m3 matrix product (no counterpart in the reference).

The steps around the matrix products of a decoder whose weights are e4m3 with
one f32 scale a row (`tans_gemv.quantize_rows`, or a decoded weight):

    q, s, h = fp8_linear.add_rms_norm_e4m3(x, weight, residual)   # h = x + residual
    y = fp8_linear.linear(q, s, w8, w_scale, bias=b, act="silu")
    q, s = fp8_linear.quantize_tokens(y)
    h = fp8_linear.linear(q, s, down8, down_scale, residual=h)

e4m3 tensors are uint8, as everywhere in this package.  All of it on sm_100a
kernels (csrc/norm.cu, csrc/linear.cu), on torch's current stream.
"""
from __future__ import annotations

import torch

from ._C import _post_check, _req, _status, _stream
from ._lib import LIB, check, on_device

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3}


def _rows(name: str, t: torch.Tensor, shape=None, dtype=None, device=None) -> int:
    """Checks [rows, cols] with a dense last dimension; the stride between rows."""
    _req(t.is_cuda and t.dim() == 2 and t.dtype in _TYPES and (t.stride(1) == 1 or t.shape[1] == 1 or not t.numel()),
         f"{name} must be a CUDA [rows, cols] bfloat16, float16 or float32 tensor with dense rows")
    if shape is not None:
        _req(t.shape == shape and t.dtype == dtype and t.device == device,
             f"{name} must have x's shape, type and device")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _norm(x, weight, residual, eps, residual_out, quantize):
    xs = _rows("x", x)
    R, C = x.shape
    dev, dt = x.device, x.dtype
    _req(weight.shape == (C,) and weight.is_contiguous() and weight.device == dev
         and weight.dtype in (dt, torch.float32), "weight must be a contiguous [cols] tensor of x's type or float32")
    rs = hs = 0
    h = residual_out
    with on_device(dev):
        if residual is not None:
            rs = _rows("residual", residual, x.shape, dt, dev)
            if h is None:
                h = torch.empty((R, C), dtype=dt, device=dev)
            hs = _rows("residual_out", h, x.shape, dt, dev)
        else:
            _req(h is None, "residual_out needs residual")
        y = q = scale = None
        if quantize:
            q = torch.empty((R, C), dtype=torch.uint8, device=dev)
            scale = torch.empty((R,), dtype=torch.float32, device=dev)
        else:
            y = torch.empty((R, C), dtype=dt, device=dev)
        check(LIB.tans_b200_add_rms_norm(
            x.data_ptr(), xs, None if residual is None else residual.data_ptr(), rs, weight.data_ptr(),
            _TYPES[weight.dtype], eps, None if h is None else h.data_ptr(), hs, None if y is None else y.data_ptr(),
            None if q is None else q.data_ptr(), None if scale is None else scale.data_ptr(), R, C, _TYPES[dt],
            _stream(dev)))
    return y, q, scale, x if h is None else h


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                 eps: float = 1e-6, residual_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual (x itself without one), y = h * rsqrt(mean(h^2)
    + eps) * weight, both [rows, cols] in x's type (bf16, f16 or f32; f32
    inside, the norm of the unrounded sum).  residual_out may be x or residual:
    then h replaces it."""
    y, _, _, h = _norm(x, weight, residual, eps, residual_out, False)
    return y, h


def add_rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                      eps: float = 1e-6, residual_out: torch.Tensor | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(q, scale, h): add_rms_norm with y as e4m3 (uint8 [rows, cols]) and one
    f32 scale a row, max|y| -> 448."""
    _, q, scale, h = _norm(x, weight, residual, eps, residual_out, True)
    return q, scale, h


def quantize_tokens(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): x [rows, cols] as e4m3 (uint8) and one f32 scale a row."""
    xs = _rows("x", x)
    R, C = x.shape
    dev = x.device
    with on_device(dev):
        q = torch.empty((R, C), dtype=torch.uint8, device=dev)
        scale = torch.empty((R,), dtype=torch.float32, device=dev)
        check(LIB.tans_b200_quantize_tokens(x.data_ptr(), xs, q.data_ptr(), scale.data_ptr(), R, C, _TYPES[x.dtype],
                                            _stream(dev)))
    return q, scale


def linear(x8: torch.Tensor, x_scale: torch.Tensor, w8: torch.Tensor, w_scale: torch.Tensor, *,
           bias: torch.Tensor | None = None, act: str = "none", mul: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """y [tokens, rows] = act(x_scale * w_scale * (x8 @ w8^T) + bias) * mul + residual.

    x8 [tokens, cols], w8 [rows, cols]: uint8 e4m3, cols a multiple of 16;
    x_scale [tokens], w_scale [rows] f32; bias [rows], mul and residual
    [tokens, rows] in the output's type (bf16 or f16).  act: "none", "relu",
    "silu" or "gelu_tanh".  f32 accumulation, one rounding.  `out` may be mul or
    residual."""
    dev = x8.device
    _req(x8.is_cuda and x8.dim() == 2 and x8.dtype == torch.uint8 and x8.is_contiguous(),
         "x8 must be a contiguous CUDA uint8 [tokens, cols] tensor of e4m3 bits")
    M, K = x8.shape
    _req(w8.dim() == 2 and w8.dtype == torch.uint8 and w8.is_contiguous() and w8.device == dev and w8.shape[1] == K,
         "w8 must be a contiguous uint8 [rows, cols] tensor of e4m3 bits with x8's columns and device")
    N = w8.shape[0]
    f32 = torch.float32
    _req(x_scale.dtype == f32 and x_scale.shape == (M,) and x_scale.is_contiguous() and x_scale.device == dev
         and w_scale.dtype == f32 and w_scale.shape == (N,) and w_scale.is_contiguous() and w_scale.device == dev,
         "x_scale must be contiguous f32 [tokens] and w_scale [rows]")
    _req(act in _ACTS, f"act must be one of {', '.join(_ACTS)}")
    _req(dtype in (torch.bfloat16, torch.float16), "dtype must be bfloat16 or float16")
    for name, t, shape in (("bias", bias, (N,)), ("mul", mul, (M, N)), ("residual", residual, (M, N)),
                           ("out", out, (M, N))):
        _req(t is None or (t.shape == shape and t.dtype == dtype and t.is_contiguous() and t.device == dev),
             f"{name} must be a contiguous {dtype} tensor of shape {shape} on x8's device")
    with on_device(dev):
        if out is None:
            out = torch.empty((M, N), dtype=dtype, device=dev)
        check(LIB.tans_b200_linear(
            x8.data_ptr(), x_scale.data_ptr(), w8.data_ptr(), w_scale.data_ptr(),
            None if bias is None else bias.data_ptr(), _ACTS[act], None if mul is None else mul.data_ptr(),
            None if residual is None else residual.data_ptr(), out.data_ptr(), M, N, K, _TYPES[dtype],
            _status(dev).data_ptr(), _stream(dev)))
    _post_check(dev)
    return out


__all__ = ["add_rms_norm", "add_rms_norm_e4m3", "quantize_tokens", "linear"]
