"""Root-mean-square norm with the residual's addition, for training (differentiable) and for serving (8-bit codes).

One CUDA kernel a call reads the two inputs once and writes the sum and the normalized rows; with the codes' form the rows leave as
8-bit codes with a scale each, as `coded_linear` reads them.  float32, bfloat16 and float16 CUDA tensors with any leading dimensions,
rows of up to 16384 elements (131071 where they are only coded); sums are held in 32 bits.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _cabi as cabi


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                 eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, total) with total = x + residual (x itself without one) and y = total * rsqrt(mean(total^2) + eps) * weight, row by row over
    the last dimension.  y is taken from the sum before it is rounded to x's type.  `weight` may be of another type than x.  Differentiable
    in x, residual and weight, once; the weight's gradient is summed in a fixed order.  Not under a trace, like the other calls here."""
    out = cabi.load_binding().add_rms_norm(x, weight, residual, eps)
    return (out[0], out[1]) if residual is not None else (out[0], x)


def add_rms_norm_codes(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
                       eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scale, total): y of `add_rms_norm` as int8 codes in [-127, 127] and a float32 scale for each row, y ~ codes * scale with
    scale = max|y| / 127.  Rows of codes start at multiples of 16 bytes.  A row of zeros has scale 0; a row with an infinity or a NaN has a
    scale that is not finite.  No gradient."""
    out = cabi.load_binding().add_rms_norm_codes(x, weight, residual, eps)
    return out[0], out[1], (out[2] if residual is not None else x)


def code_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of the rows of x as they are, in the form of `add_rms_norm_codes`."""
    out = cabi.load_binding().add_rms_norm_codes(x, None, None, 0.0)
    return out[0], out[1]
