"""Root-mean-square norm with the residual's addition and an 8-bit result: what stands before every projection of a
transformer block whose weights are quantised.  One kernel (csrc/norm.cu) reads x and the residual once and writes the new
residual, the quantised rows and their scales, which `linear(..., act_scale=...)` multiplies.  The reference has no counterpart
in its GEMM path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .gemm_kernels import Scalar
from .quantize import _as_2d, _check_row_cols

_FORMATS = {None: _lib.NORM_NONE, "int8": _lib.NORM_INT8, "fp8_block128": _lib.NORM_FP8_GROUP_1X128, "fp8": _lib.NORM_FP8_GIVEN}


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
             format: Optional[str] = None, scale: Scalar = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """x [..., K] (float32 / bfloat16 / float16) -> (result, scales, x + residual).

        t = x + residual, rounded to the type of x  (without a residual t = x, and the third result is None)
        y = t * rsqrt(mean(t^2) + eps) * weight     (fp32)

    `format` names the packed-weight format of the projection that reads the result:
    * None            the result is y in the type and shape of x, no scales
    * "int8"          int8 [rows, K], scales fp32 [rows]: `quantize_int8` of y
    * "fp8_block128"  E4M3 bytes uint8 [rows, K], scales fp32 [rows, ceil(K/128)]: `quantize_fp8(y, "groupwise")`
    * "fp8"           E4M3 bytes with the given per-tensor `scale` (a calibrated one: a number or a one-element tensor; taking the
                      maximum of the whole tensor would cost a second pass): `quantize_fp8(y, scale=scale)`; scales is that scale
    Hand result and scales to `linear(result, packed, act_scale=scales)`.  `weight` [K] may have a type of its own.  K must be a
    multiple of 16, at most 32768.  A row with a NaN or an infinity is NaN throughout or as IEEE arithmetic has it; no other row is
    touched.
    """
    if format not in _FORMATS:
        raise ValueError(f"format must be None, 'int8', 'fp8_block128' or 'fp8', got {format!r}")
    if (scale is not None) != (format == "fp8"):
        raise ValueError("format 'fp8' needs the scale of the result; the other formats derive theirs")
    dev = _lib.require_cuda(x, weight, residual)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have at least one element in its last dimension, got {tuple(x.shape)}")
    cols = x.shape[-1]
    _check_row_cols(cols)
    if weight.dim() != 1 or weight.shape[0] != cols:
        raise ValueError(f"weight must be [{cols}], got {tuple(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have the shape and type of x, got {tuple(residual.shape)} {residual.dtype}")
    x2 = x if x.dim() == 2 and x.is_contiguous() else _as_2d(x)
    rows = x2.shape[0]
    weight = weight.contiguous()
    r2 = total = s = s_in = None                              # (empty_like takes half of the host time of torch.empty)
    if residual is not None:
        r2 = residual if residual.dim() == 2 and residual.is_contiguous() else _as_2d(residual)
        total = torch.empty_like(x) if x2 is x else torch.empty_like(x2).view(x.shape)
    if format is None:
        out = torch.empty_like(x) if x2 is x else torch.empty_like(x2).view(x.shape)
    else:
        out = torch.empty_like(x2, dtype=torch.int8 if format == "int8" else torch.uint8)
    if format == "int8":
        s = torch.empty(rows, dtype=torch.float32, device=dev)
    elif format == "fp8_block128":
        groups = (cols + 127) // 128
        s = torch.empty_strided((rows, groups), (groups, 1), dtype=torch.float32, device=dev)
    elif format == "fp8":
        s = s_in = (scale.detach().to(device=dev, dtype=torch.float32).reshape(1) if isinstance(scale, torch.Tensor)
                    else torch.full((1,), float(scale), dtype=torch.float32, device=dev))
    if rows == 0:                       # an empty tensor has no address
        return out, s, total
    with _lib.on_device(dev):
        rc = _lib.lib().dsl_rms_norm(x2.data_ptr(), _lib.dtype_code(x2.dtype), rows, cols, _lib.ptr(r2), weight.data_ptr(),
                                     _lib.dtype_code(weight.dtype), eps, _FORMATS[format], _lib.ptr(total), out.data_ptr(), _lib.ptr(s),
                                     _lib.ptr(s_in), _lib.stream_ptr(dev.index))
    _lib.check(rc, "dsl_rms_norm")
    return out, s, total
