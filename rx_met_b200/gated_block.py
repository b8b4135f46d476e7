"""A block of a streaming model on the gated recurrence: training with activations kept in 8 bits, serving in 8-bit codes.

    f, v, g = norm(x) W_in        h = x + (silu(g) * recurrence(f, v)) W_mix        y = h + (silu(a) * b) W_down,   a, b = norm(h) W_up

`GatedBlock` trains in 16 or 32 bits.  What its backward pass needs of an activation is kept as codes: the inputs of its four products, and both factors of its two gated products; only the gates and the
values of the recurrence are kept as they are.  `GatedBlock.coded()` serves it as `DecayBlock.coded()` does: a prompt goes through `prefill`, further tokens one by one through `step`, which
updates the state in place.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .coded_linear import code_weight, coded_linear
from .gated_recurrence import gated_recurrence, gated_recurrence_step
from .kept_codes import gated_product, linear
from .rms_norm import add_rms_norm, add_rms_norm_codes, code_rows


class GatedBlock(torch.nn.Module):
    """width: of the stream; inner: channels of the recurrence; hidden: of the second half.  The memories of the channels are spread from two tokens to `longest`."""

    def __init__(self, width: int, inner: int, hidden: int, longest: float = 512.0, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        make = lambda rows, cols: torch.nn.Parameter((torch.randn(rows, cols, device=device) * cols ** -0.5).to(dtype))  # noqa: E731
        self.norm1 = torch.nn.Parameter(torch.ones(width, device=device))
        self.norm2 = torch.nn.Parameter(torch.ones(width, device=device))
        self.w_in, self.w_mix, self.w_up, self.w_down = make(3 * inner, width), make(width, inner), make(2 * hidden, width), make(width, hidden)
        # sigmoid(bias) = 1 - 1 / memory
        memories = torch.logspace(0.30103, float(torch.tensor(longest).log10()), inner, device=device)
        self.bias = torch.nn.Parameter(torch.cat([torch.log(memories - 1), torch.zeros(2 * inner, device=device)]).to(dtype))

    @property
    def dtype(self) -> torch.dtype:
        return self.w_in.dtype

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(y, final state [batch, inner]) of x [batch, tokens, width], differentiable."""
        y, _ = add_rms_norm(x, self.norm1)
        forget, value, gate = linear(y, self.w_in, self.bias).chunk(3, dim=-1)
        out, last = gated_recurrence(forget, value, state=state, lengths=lengths)
        y, h = add_rms_norm(linear(gated_product(gate, out), self.w_mix), self.norm2, x)
        a, b = linear(y, self.w_up).chunk(2, dim=-1)
        return h + linear(gated_product(a, b), self.w_down), last

    def coded(self) -> "CodedGatedBlock":
        return CodedGatedBlock(self)


class CodedGatedBlock:
    """The block with 8-bit weights and 8-bit codes in front of every product, as the block is when this is made: it keeps copies of all its values.  No gradients."""

    def __init__(self, block: GatedBlock):
        self.dtype = block.dtype
        self.w_in, self.w_mix, self.w_up, self.w_down = (code_weight(w) for w in (block.w_in, block.w_mix, block.w_up, block.w_down))
        self.norm1, self.norm2, self.bias = (t.detach().clone() for t in (block.norm1, block.norm2, block.bias.float()))

    def _around(self, x, mix):
        codes, scale, _ = add_rms_norm_codes(x, self.norm1)
        forget, value, gate = coded_linear(codes, scale, self.w_in, bias=self.bias, dtype=self.dtype).chunk(3, dim=-1)
        h = coded_linear(*code_rows(gated_product(gate, mix(forget, value))), self.w_mix, residual=x, dtype=self.dtype)
        codes, scale, _ = add_rms_norm_codes(h, self.norm2)
        a, b = coded_linear(codes, scale, self.w_up, dtype=self.dtype).chunk(2, dim=-1)
        return coded_linear(*code_rows(gated_product(a, b)), self.w_down, residual=h, dtype=self.dtype)

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(y, final state) of x [batch, tokens, width]."""
        last = []

        def mix(forget, value):
            out, final = gated_recurrence(forget, value, state=state, lengths=lengths)
            last.append(final)
            return out

        y = self._around(x, mix)
        return y, last[0]

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, active: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y of one token for each row, x [batch, width]; `state` is updated in place."""
        return self._around(x, lambda forget, value: gated_recurrence_step(forget, value, state, active=active))
