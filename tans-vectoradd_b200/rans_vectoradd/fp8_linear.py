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

from ._C import _post_check, _status
from ._lib import LIB, check, on_device, ptr, raw_stream

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3}


def _stride(name: str, t: torch.Tensor, cols: int) -> int:
    """The stride between the rows of a two-dimensional t whose last dimension must be dense."""
    if t.is_contiguous():
        return cols
    st = t.stride()
    if st[1] != 1 and cols != 1:
        raise RuntimeError(f"{name} must have dense rows")
    return st[0]


def _rows(name: str, t: torch.Tensor) -> tuple[torch.Size, int]:
    """Checks [rows, cols] with a dense last dimension: its shape, the stride between rows."""
    shape = t.shape
    if len(shape) != 2 or t.dtype not in _TYPES or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA [rows, cols] bfloat16, float16 or float32 tensor")
    return shape, _stride(name, t, shape[1])


def _like_x(name: str, t: torch.Tensor, shape: torch.Size, dtype: torch.dtype, dev: torch.device) -> int:
    if t.shape != shape or t.dtype != dtype or t.device != dev:
        raise RuntimeError(f"{name} must have x's shape, type and device")
    return _stride(name, t, shape[1])


def _norm(x, weight, residual, eps, residual_out, quantize):
    shape, xs = _rows("x", x)
    R, C = shape
    dev, dt, wt = x.device, x.dtype, weight.dtype
    if (weight.shape != (C,) or not weight.is_contiguous() or weight.device != dev
            or (wt != dt and wt != torch.float32)):
        raise RuntimeError("weight must be a contiguous [cols] tensor of x's type or float32")
    rs = hs = 0
    h, r_ptr, h_ptr = x, None, None
    with on_device(dev):
        if residual is not None:
            rs, r_ptr = _like_x("residual", residual, shape, dt, dev), residual.data_ptr()
            if residual_out is None:
                h, hs = torch.empty(R, C, dtype=dt, device=dev), C
            else:
                h, hs = residual_out, _like_x("residual_out", residual_out, shape, dt, dev)
            h_ptr = h.data_ptr()
        elif residual_out is not None:
            raise RuntimeError("residual_out needs residual")
        if quantize:
            y = torch.empty(R, C, dtype=torch.uint8, device=dev)
            scale = torch.empty(R, dtype=torch.float32, device=dev)
            y_ptr, q_ptr, s_ptr = None, y.data_ptr(), scale.data_ptr()
        else:
            y, scale = torch.empty(R, C, dtype=dt, device=dev), None
            y_ptr, q_ptr, s_ptr = y.data_ptr(), None, None
        check(LIB.tans_b200_add_rms_norm(x.data_ptr(), xs, r_ptr, rs, weight.data_ptr(), _TYPES[wt], eps, h_ptr, hs,
                                         y_ptr, q_ptr, s_ptr, R, C, _TYPES[dt], raw_stream(dev)))
    return y, scale, h


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                 eps: float = 1e-6, residual_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h): h = x + residual (x itself without one), y = h * rsqrt(mean(h^2)
    + eps) * weight, both [rows, cols] in x's type (bf16, f16 or f32; f32
    inside, the norm of the unrounded sum).  residual_out may be x or residual:
    then h replaces it."""
    y, _, h = _norm(x, weight, residual, eps, residual_out, False)
    return y, h


def add_rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                      eps: float = 1e-6, residual_out: torch.Tensor | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(q, scale, h): add_rms_norm with y as e4m3 (uint8 [rows, cols]) and one
    f32 scale a row, max|y| -> 448."""
    return _norm(x, weight, residual, eps, residual_out, True)


def quantize_tokens(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): x [rows, cols] as e4m3 (uint8) and one f32 scale a row."""
    (R, C), xs = _rows("x", x)
    dev = x.device
    with on_device(dev):
        q = torch.empty(R, C, dtype=torch.uint8, device=dev)
        scale = torch.empty(R, dtype=torch.float32, device=dev)
        check(LIB.tans_b200_quantize_tokens(x.data_ptr(), xs, q.data_ptr(), scale.data_ptr(), R, C, _TYPES[x.dtype],
                                            raw_stream(dev)))
    return q, scale


def _check_operand(name, t, shape, dtype, dev):
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.device != dev:
        raise RuntimeError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on x8's device")


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
    if not x8.is_cuda or x8.dim() != 2 or x8.dtype != torch.uint8 or not x8.is_contiguous():
        raise RuntimeError("x8 must be a contiguous CUDA uint8 [tokens, cols] tensor of e4m3 bits")
    M, K = x8.shape
    if (w8.dim() != 2 or w8.dtype != torch.uint8 or not w8.is_contiguous() or w8.device != dev
            or w8.shape[1] != K):
        raise RuntimeError("w8 must be a contiguous uint8 [rows, cols] tensor of e4m3 bits with x8's columns and device")
    N = w8.shape[0]
    f32 = torch.float32
    if (x_scale.dtype != f32 or x_scale.shape != (M,) or not x_scale.is_contiguous() or x_scale.device != dev
            or w_scale.dtype != f32 or w_scale.shape != (N,) or not w_scale.is_contiguous() or w_scale.device != dev):
        raise RuntimeError("x_scale must be contiguous f32 [tokens] and w_scale [rows]")
    if act not in _ACTS:
        raise RuntimeError(f"act must be one of {', '.join(_ACTS)}")
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise RuntimeError("dtype must be bfloat16 or float16")
    if bias is not None:
        _check_operand("bias", bias, (N,), dtype, dev)
    if mul is not None:
        _check_operand("mul", mul, (M, N), dtype, dev)
    if residual is not None:
        _check_operand("residual", residual, (M, N), dtype, dev)
    if out is not None:
        _check_operand("out", out, (M, N), dtype, dev)
    with on_device(dev):
        if out is None:
            out = torch.empty(M, N, dtype=dtype, device=dev)
        check(LIB.tans_b200_linear(
            x8.data_ptr(), x_scale.data_ptr(), w8.data_ptr(), w_scale.data_ptr(),
            ptr(bias), _ACTS[act], ptr(mul), ptr(residual), out.data_ptr(), M, N, K, _TYPES[dtype],
            _status(dev).data_ptr(), raw_stream(dev)))
    _post_check(dev)
    return out


__all__ = ["add_rms_norm", "add_rms_norm_e4m3", "quantize_tokens", "linear"]
