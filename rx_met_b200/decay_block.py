"""A block of a streaming model on linear attention with decays: what the three operators of the token mixer look like together.

    h = x + attention(norm(x)) W_out        y = h + silu(norm(h) W_up + b_up) W_down

`DecayBlock` trains in 16 or 32 bits: its norms and its attention are this package's differentiable kernels, its four products torch's.  `DecayBlock.coded()`
serves it: the norms leave 8-bit codes, the products are taken on them, and bias, activation and residual are applied where the sums leave the tensor
cores.  A prompt goes through `CodedDecayBlock.prefill`, further tokens one by one through `step`, which updates the state in place.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from .coded_linear import code_weight, coded_linear
from .decayed_attention import decayed_attention, decayed_attention_step
from .rms_norm import add_rms_norm, add_rms_norm_codes, code_rows


class DecayBlock(torch.nn.Module):
    """width: of the stream; heads of head_dim elements; hidden: of the second half.  The memories of the heads are spread from two tokens to `longest`."""

    def __init__(self, width: int, heads: int, head_dim: int, hidden: int, longest: float = 512.0, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.heads, self.head_dim = heads, head_dim
        inner = heads * head_dim
        make = lambda rows, cols: torch.nn.Parameter((torch.randn(rows, cols, device=device) * cols ** -0.5).to(dtype))  # noqa: E731
        self.norm1 = torch.nn.Parameter(torch.ones(width, device=device))
        self.norm2 = torch.nn.Parameter(torch.ones(width, device=device))
        self.w_qkv, self.w_out, self.w_up, self.w_down = make(3 * inner, width), make(width, inner), make(hidden, width), make(width, hidden)
        self.b_up = torch.nn.Parameter(torch.zeros(hidden, device=device))
        self.register_buffer("log_decay", torch.log1p(-1 / torch.logspace(0.30103, float(torch.tensor(longest).log10()), heads, device=device)))

    @property
    def dtype(self) -> torch.dtype:
        return self.w_qkv.dtype

    def _apply(self, fn, recurse=True):
        """to() and its kind: the decays stay in 32 bits, whose exponents the heads with long memories need."""
        kept = self.log_decay
        super()._apply(fn, recurse)
        self.log_decay = kept.to(self.log_decay.device)
        return self

    def _split(self, qkv):
        return (t.unflatten(-1, (self.heads, self.head_dim)) for t in qkv.chunk(3, dim=-1))

    def forward(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(y, final state) of x [batch, tokens, width], differentiable."""
        y, _ = add_rms_norm(x, self.norm1)
        out, last = decayed_attention(*self._split(F.linear(y, self.w_qkv)), self.log_decay, state=state, lengths=lengths)
        y, h = add_rms_norm(F.linear(out.flatten(2), self.w_out), self.norm2, x)
        return h + F.linear(F.silu(F.linear(y, self.w_up, self.b_up.to(self.dtype))), self.w_down), last

    def coded(self) -> "CodedDecayBlock":
        return CodedDecayBlock(self)


class CodedDecayBlock:
    """The block with 8-bit weights and 8-bit codes in front of every product, as the block is when this is made: it keeps copies of all its values.  No gradients."""

    def __init__(self, block: DecayBlock):
        self.heads, self.head_dim, self.dtype = block.heads, block.head_dim, block.dtype
        self.qkv, self.out, self.up, self.down = (code_weight(w) for w in (block.w_qkv, block.w_out, block.w_up, block.w_down))
        self.norm1, self.norm2, self.b_up, self.log_decay = (t.detach().clone() for t in (block.norm1, block.norm2, block.b_up.float(), block.log_decay))

    def _around(self, x, attend):
        codes, scale, _ = add_rms_norm_codes(x, self.norm1)
        qkv = coded_linear(codes, scale, self.qkv, dtype=self.dtype)
        out = attend(*(t.unflatten(-1, (self.heads, self.head_dim)) for t in qkv.chunk(3, dim=-1)))
        h = coded_linear(*code_rows(out.flatten(-2)), self.out, residual=x, dtype=self.dtype)
        codes, scale, _ = add_rms_norm_codes(h, self.norm2)
        up = coded_linear(codes, scale, self.up, bias=self.b_up, activation="silu", dtype=self.dtype)
        return coded_linear(*code_rows(up), self.down, residual=h, dtype=self.dtype)

    @torch.no_grad()
    def prefill(self, x: torch.Tensor, state: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(y, final state) of x [batch, tokens, width]."""
        last = []

        def attend(q, k, v):
            out, final = decayed_attention(q, k, v, self.log_decay, state=state, lengths=lengths)
            last.append(final)
            return out

        y = self._around(x, attend)
        return y, last[0]

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, active: Optional[torch.Tensor] = None) -> torch.Tensor:
        """y of one token for each row, x [batch, width]; `state` is updated in place."""
        return self._around(x, lambda q, k, v: decayed_attention_step(q, k, v, self.log_decay, state, active=active))
