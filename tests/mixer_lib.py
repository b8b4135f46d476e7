"""Plain forms of the token mixer's operators in 64 bits, and bounds on the errors of the 32-bit and 16-bit ones (test infrastructure)."""
from __future__ import annotations

import math

import torch

#: half a unit in the last place, relative
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
#: half of the smallest step, absolute
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def within(got, want, bound):
    """Every element of `got` within `bound` of `want` (tensors of 64 bits, `bound` as `want`); a message that names the worst one."""
    got, off = got.double(), (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()), "not finite"
    if off.numel():
        worst = (off - bound).argmax()
        assert bool((off <= bound).all()), f"off by {off.flatten()[worst]:.3e}, allowed {bound.flatten()[worst]:.3e}, value {want.flatten()[worst]:.3e}"


def norm(x, weight, residual, eps):
    total = x.double() + (residual.double() if residual is not None else 0)
    rms = torch.rsqrt((total ** 2).mean(dim=-1, keepdim=True) + eps)
    return total * rms * weight.double(), total, rms


def norm_gradients(dy, dtotal, total, weight, rms):
    u, d = total * rms, dy.double() * weight.double()
    dx = rms * (d - u * (d * u).mean(dim=-1, keepdim=True))
    return (dx if dtotal is None else dx + dtotal.double()), (dy.double() * u).flatten(0, -2).sum(dim=0)


def linear(codes, scale, weight, weight_scale, bias, activation, residual):
    """(value, magnitude): magnitude is what the roundings in front of the activation are relative to."""
    y = (codes.double() @ weight.double().T) * scale.double()[..., None] * weight_scale.double()
    z = y if bias is None else y + bias.double()
    magnitude = y.abs() + (0 if bias is None else bias.double().abs())
    out = {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))}[activation](z)
    if residual is not None:
        out, magnitude = out + residual.double(), magnitude + residual.double().abs()
    return out, magnitude


def attend(q, k, v, log_decay, state, lengths, scale):
    """(out, final state), token by token."""
    B, T = q.shape[:2]
    H = log_decay.numel()
    q, k, v = (t.double().repeat_interleave(H // t.shape[2], dim=2) for t in (q, k, v))
    decay = torch.exp(log_decay.double())[:, None, None]
    S = torch.zeros(B, H, q.shape[3], v.shape[3], dtype=torch.float64, device=q.device) if state is None else state.double()
    out = torch.zeros(B, T, H, v.shape[3], dtype=torch.float64, device=q.device)
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool, device=q.device) if lengths is None else t < lengths.to(q.device)
        at = live[:, None, None]
        kt, vt, qt = (torch.where(at, x[:, t], torch.zeros_like(x[:, t])) for x in (k, v, q))   # padding may hold anything
        S = torch.where(at[..., None], decay * S + kt[..., None] * vt[..., None, :], S)
        out[:, t] = (qt[..., None, :] @ S)[..., 0, :] * scale
    return out, S


def attend_gradients(q, k, v, log_decay, state, lengths, scale, dout, dfinal):
    """Gradients of q, k, v and state by the recurrence of the state's gradient, from the last token to the first."""
    B, T = q.shape[:2]
    H = log_decay.numel()
    heads = [t.shape[2] for t in (q, k, v)]
    q, k, v = (t.double().repeat_interleave(H // t.shape[2], dim=2) for t in (q, k, v))
    decay = torch.exp(log_decay.double())[:, None, None]
    S = torch.zeros(B, H, q.shape[3], v.shape[3], dtype=torch.float64, device=q.device) if state is None else state.double()
    G = torch.zeros_like(S) if dfinal is None else dfinal.double()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    masked = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool, device=q.device) if lengths is None else t < lengths.to(q.device)
        at = live[:, None, None]
        rows = [torch.where(at, x[:, t], torch.zeros_like(x[:, t])) for x in (q, k, v, dout.double())]
        masked.append((at, rows))
        S = torch.where(at[..., None], decay * S + rows[1][..., None] * rows[2][..., None, :], S)
        dq[:, t] = (S @ rows[3][..., None])[..., 0] * scale
    for t in reversed(range(T)):
        at, (qt, kt, vt, dt) = masked[t]
        new = G + qt[..., None] * dt[..., None, :] * scale
        dk[:, t] = (new @ vt[..., None])[..., 0]
        dv[:, t] = (kt[..., None, :] @ new)[..., 0, :]
        G = torch.where(at[..., None], decay * new, G)
    group = lambda d, n: d.view(B, T, n, H // n, -1).sum(dim=3)  # noqa: E731
    return group(dq, heads[0]), group(dk, heads[1]), group(dv, heads[2]), G


def magnitudes(function, tensors, *rest):
    """The same function of the magnitudes: what its rounding errors are relative to."""
    return function(*(t if t is None else t.abs() for t in tensors), *rest)


def attention_bound(magnitude, dtype, tokens, dim, out_type):
    """Error of an output of `magnitude`: 32-bit sums over tokens and a head's elements, each step off by two roundings at most, and
    a power of the decay by as many as its exponent; with 16-bit inputs products on tensor cores take one of their operands rounded to that type (float16:
    by half of its smallest step at least, times inputs below 5, for the tokens of a part and the elements of a head).  Then the rounding to `out_type`."""
    sums = (4 * tokens + 2 * dim + 32) * 2.0 ** -24
    operand = 0.0 if dtype == torch.float32 else UNIT[dtype]
    unit = UNIT[out_type]
    return magnitude * ((1 + sums + operand * 1.01) * (1 + unit) - 1) + TINY[out_type] + (0 if dtype != torch.float16 else (dim + min(tokens, 128)) * 2.0 ** -25 * 5)
