"""The token mixer's plain forms agree with one another, and its entry points refuse tensors that are not on a GPU."""
import pytest
import torch

import mixer_lib as ml


def test_gradients_of_the_plain_forms():
    """The recurrences written for the gradients against automatic differentiation of the forward recurrence."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 9, h, d, generator=g, dtype=torch.float64).requires_grad_() for h, d in ((4, 5), (2, 5), (1, 3)))
    state = torch.randn(2, 4, 5, 3, generator=g, dtype=torch.float64).requires_grad_()
    decay, lengths = torch.tensor([0.0, -0.1, -1.0, -20.0]), torch.tensor([9, 4])
    dout, dlast = torch.randn(2, 9, 4, 3, generator=g, dtype=torch.float64), torch.randn(2, 4, 5, 3, generator=g, dtype=torch.float64)
    head = lambda t: t.repeat_interleave(4 // t.shape[2], dim=2)  # noqa: E731
    S, outs = state, []
    for t in range(9):
        live = (t < lengths)[:, None, None].double()
        new = torch.exp(decay.double())[:, None, None] * S + head(k)[:, t, :, :, None] * head(v)[:, t, :, None, :]
        S = torch.where(live[..., None] > 0, new, S)
        outs.append((head(q)[:, t, :, None, :] @ S)[..., 0, :] * 0.7 * live)
    grads = torch.autograd.grad([torch.stack(outs, dim=1), S], [q, k, v, state], [dout, dlast])
    wants = ml.attend_gradients(q.detach(), k.detach(), v.detach(), decay, state.detach(), lengths, 0.7, dout, dlast)
    for got, want in zip(grads, wants):
        assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    out, last = ml.attend(q.detach(), k.detach(), v.detach(), decay, state.detach(), lengths, 0.7)
    assert torch.allclose(out, torch.stack(outs, dim=1)) and torch.allclose(last, S)


def test_norm_gradient_of_the_plain_form():
    g = torch.Generator().manual_seed(1)
    x, residual = (torch.randn(3, 7, generator=g, dtype=torch.float64).requires_grad_() for _ in range(2))
    weight = torch.randn(7, generator=g, dtype=torch.float64).requires_grad_()
    dy, dtotal = torch.randn(3, 7, generator=g, dtype=torch.float64), torch.randn(3, 7, generator=g, dtype=torch.float64)
    y, total, rms = ml.norm(x, weight, residual, 1e-3)
    grads = torch.autograd.grad([y, total], [x, residual, weight], [dy, dtotal])
    dx, dweight = ml.norm_gradients(dy, dtotal, total.detach(), weight.detach(), rms.detach())
    assert torch.allclose(grads[0], dx) and torch.allclose(grads[1], dx) and torch.allclose(grads[2], dweight)


def test_tensors_off_the_gpu_are_refused():
    from rx_met_b200 import coded_linear, decayed_attention, rms_norm
    x = torch.zeros(2, 16)
    q = torch.zeros(1, 2, 1, 16)
    for call in (lambda: rms_norm.add_rms_norm(x, torch.ones(16)), lambda: rms_norm.add_rms_norm_codes(x, torch.ones(16)), lambda: rms_norm.code_rows(x),
                 lambda: coded_linear.coded_linear(x.to(torch.int8), torch.ones(2), coded_linear.CodedWeight(x.to(torch.int8), torch.ones(2))),
                 lambda: decayed_attention.decayed_attention(q, q, q, torch.zeros(1)),
                 lambda: decayed_attention.decayed_attention_step(q[0], q[0], q[0], torch.zeros(1), torch.zeros(2, 1, 16, 16))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
