"""Linear layers in 8-bit integers: the product with a scale for each token and each output channel, and the two
producers of its operands, quantisation by rows and the root-mean-square norm that ends in it.  (The per-tensor e4m3
counterparts are ``fp8_gemm_scaled`` and ``fp8_quantize_per_tensor``.)  For inference: no result carries a gradient."""
from __future__ import annotations

import torch

from .ops import add_rms_norm_int8_call, int8_gemm_call, int8_quantize_call, rms_norm_int8_call


def int8_gemm(x: torch.Tensor, y: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, *, bias: torch.Tensor | None = None,
              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``out[m, n] = cast(sum_k x[m, k] * y[k, n] * scale_a[m] * scale_b[n] + bias[n])``.

    x: [m, k] int8, y: [k, n] int8 with any strides; ``w.t()`` of a contiguous [n, k] weight with ``k % 16 == 0`` is the fast
    layout (both operands are read in place; others are copied into a workspace first).  The sum is exact (``k <= 131071``); scales (float32, m and n elements in any shape) and bias (n elements of float16, bfloat16 or
    float32) are applied in fp32.  out_dtype: float16, bfloat16 or float32."""
    return int8_gemm_call(x, y, scale_a, scale_b, bias, out_dtype)


def int8_quantize_per_token(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)`` with ``q * scale ~ x``: for each row of the last dimension (1 to 65536 elements) ``scale = max|x| / 127``
    (1 for a row of zeros) and ``q = round(x * 127 / max|x|)``, ties to even.  x: float16, bfloat16 or float32 of any shape;
    q has its shape in int8, scale is ``[..., 1]`` float32.  A row with a NaN or an infinity gets that as its scale and zeros
    as its integers.  The rows of an [n, k] weight are the output channels: ``wq, ws = int8_quantize_per_token(w)`` and
    ``int8_gemm(q, wq.t(), scale, ws)``."""
    return int8_quantize_call(x)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                  eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor] | tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Root-mean-square norm over the last dimension with 8-bit output: ``(q, scale)`` of
    ``h * rsqrt(mean(h^2) + eps) * weight`` as in :func:`int8_quantize_per_token`, with ``h = x``; or, with a residual of x's
    shape, ``(q, scale, h)`` with ``h = x + residual`` rounded to x's dtype: the new residual, of whose rounded values the
    norm is taken.  weight: [width] of x's dtype.  The mean of the squares is fp64; the integers are those of the formula for 16-bit
    types (for float32 ``h * weight`` is rounded once), the scale is rounded once."""
    if residual is None:
        return rms_norm_int8_call(x, weight, eps)
    return add_rms_norm_int8_call(x, residual, weight, eps)
