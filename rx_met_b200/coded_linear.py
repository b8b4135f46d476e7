"""Product of 8-bit codes with 8-bit weights; bias, activation and residual are applied where the sums leave the tensor cores.

The sums are exact in 32-bit integers, as in the recurrent layers; scales belong to rows of the input and to output channels.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _cabi as cabi
from .rms_norm import code_rows

#: activations by name, as the library numbers them
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class CodedWeight(NamedTuple):
    """A weight [outer, inner] as int8 codes and a float32 scale for each of its rows.  Rows of `codes` should start at multiples of 16
    bytes, as those of `code_weight` do; others are taken, by a slower kernel."""
    codes: torch.Tensor
    scale: torch.Tensor


def code_weight(weight: torch.Tensor) -> CodedWeight:
    """Codes of a weight [outer, inner] with a symmetric 8-bit grid for each output channel.  Once a weight, not once a call."""
    if weight.dim() != 2:
        raise RuntimeError("code_weight takes a weight of two dimensions, [outer, inner]")
    return CodedWeight(*code_rows(weight.detach()))


def coded_linear(codes: torch.Tensor, scale: torch.Tensor, weight: CodedWeight, *, bias: Optional[torch.Tensor] = None,
                 activation: str = "none", residual: Optional[torch.Tensor] = None,
                 dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """activation((codes @ weight.codes.T) * scale * weight.scale + bias) + residual in `dtype` (float32, bfloat16 or float16).
    codes int8 [..., inner], scale float32 [...], bias float32 [outer], residual of `dtype` [..., outer].  gelu is the erf form.  inner is at most
    131071, the numbers of rows and of outer channels at most 4194240 each.  No gradient."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"coded_linear: activation {activation!r}, one of {', '.join(ACTIVATIONS)}")
    if dtype not in _TYPES:
        raise RuntimeError(f"coded_linear: output type {dtype}, one of float32, bfloat16, float16")
    return cabi.load_binding().coded_linear(codes, scale, weight.codes, weight.scale, bias, ACTIVATIONS[activation], residual,
                                            _TYPES[dtype])
