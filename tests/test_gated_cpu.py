"""The gated mixer's plain forms agree with one another, and its entry points refuse what needs no GPU to be refused."""
import pytest
import torch

import gated_lib as gl


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("activation", ["none", "tanh"])
def test_gradients_of_the_plain_recurrence(own, activation):
    """The recurrence written for the gradients against automatic differentiation of the forward recurrence."""
    g = torch.Generator().manual_seed(0)
    make = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float64)  # noqa: E731
    forget, value, state = (t.requires_grad_() for t in (make(3, 9, 5), make(3, 9, 5), make(3, 5)))
    input = make(3, 9, 5).requires_grad_() if own else None
    lengths, dout, dfinal = torch.tensor([9, 0, 4]), make(3, 9, 5), make(3, 5)
    f = torch.sigmoid(forget)
    z = 1 - f if input is None else torch.sigmoid(input)
    c = torch.tanh(value) if activation == "tanh" else value
    h, outs = state, []
    for t in range(9):
        live = (t < lengths)[:, None]
        h = torch.where(live, f[:, t] * h + z[:, t] * c[:, t], h)
        outs.append(h * live)
    leaves = [t for t in (forget, value, input, state) if t is not None]
    grads = torch.autograd.grad([torch.stack(outs, dim=1), h], leaves, [dout, dfinal])
    plain = [t.detach() if t is not None else None for t in (forget, value, input)]
    wants = gl.recur_gradients(*plain, activation, state.detach(), lengths, dout, dfinal)
    for got, want in zip(grads, [w for w in wants if w is not None]):
        assert torch.allclose(got, want[0], rtol=1e-12, atol=1e-12)
    out, last, *_ = gl.recur(*plain, activation, state.detach(), lengths)
    assert torch.allclose(out, torch.stack(outs, dim=1)) and torch.allclose(last, h)


def test_tensors_off_the_gpu_are_refused():
    from rx_met_b200 import gated_recurrence
    x = torch.zeros(2, 3, 16)
    for call in (lambda: gated_recurrence.gated_recurrence(x, x), lambda: gated_recurrence.gated_recurrence_step(x[:, 0], x[:, 0], torch.zeros(2, 16))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="activation"):
        gated_recurrence.gated_recurrence(x, x, activation="relu")
