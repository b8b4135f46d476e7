"""The token mixer's operators together: a block that trains in floats and serves in 8-bit codes."""
import pytest
import torch
import torch.nn.functional as F

import mixer_lib as ml

pytestmark = pytest.mark.gpu


def block(dtype, seed=0):
    from rx_met_b200.decay_block import DecayBlock
    torch.manual_seed(seed)
    return DecayBlock(width=192, heads=4, head_dim=48, hidden=400, dtype=dtype)


def eager(b, x, state, lengths):
    """The block in 64 bits."""
    w = {n: p.detach().double() for n, p in b.named_parameters()}
    norm = lambda t, s: t * torch.rsqrt((t ** 2).mean(dim=-1, keepdim=True) + 1e-6) * s  # noqa: E731
    q, k, v = (t.unflatten(-1, (b.heads, b.head_dim)) for t in F.linear(norm(x.double(), w["norm1"]), w["w_qkv"]).chunk(3, dim=-1))
    out, last = ml.attend(q, k, v, b.log_decay, state, lengths, b.head_dim ** -0.5)
    h = x.double() + F.linear(out.flatten(2), w["w_out"])
    return h + F.linear(F.silu(F.linear(norm(h, w["norm2"]), w["w_up"], w["b_up"])), w["w_down"]), last


def off(got, want):
    return float((got.detach().double() - want).norm() / want.norm())


# relative, over the whole output: six roundings of 2^-9 to 2^-8 of their type's values in a row for 16 bits; 8-bit codes of four products are off by 127^-1 / sqrt(12) of a row's largest
# value, about four times its mean
@pytest.mark.parametrize("dtype,floats,codes", [(torch.float32, 1e-5, 0.05), (torch.bfloat16, 0.02, 0.05), (torch.float16, 0.003, 0.05)])
def test_block_against_its_formula(dtype, floats, codes):
    b = block(dtype)
    x = torch.randn(3, 150, 192, device="cuda").to(dtype)
    state = torch.randn(3, 4, 48, 48, device="cuda")
    lengths = torch.tensor([150, 0, 77], device="cuda")
    want, wanted_last = eager(b, x, state, lengths)
    y, last = b(x, state, lengths)
    assert off(y, want) < floats and off(last, wanted_last) < floats
    y, last = b.coded().prefill(x, state, lengths)
    assert y.dtype == dtype and off(y, want) < codes and off(last, wanted_last) < codes


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_prompt_and_its_tokens(dtype):
    """A prompt at once, and its last tokens one by one behind the rest of it."""
    c = block(dtype, seed=1).coded()
    x = torch.randn(2, 140, 192, device="cuda").to(dtype)
    whole, last = c.prefill(x)
    first, state = c.prefill(x[:, :132])
    tail = torch.stack([c.step(x[:, t], state) for t in range(132, 140)], dim=1)
    # the two ways round differently, and a code may fall on the other side of a half
    assert off(tail, whole[:, 132:].double()) < 0.02 and off(state, last.double()) < 0.02 and torch.isfinite(tail).all()
    assert off(first, whole[:, :132].double()) < 0.02


def test_block_trains():
    """Gradients of all parameters against automatic differentiation of the formula in 64 bits, and a step along them."""
    b = block(torch.float32, seed=2)
    x = torch.randn(2, 40, 192, device="cuda")
    target = torch.randn(2, 40, 192, device="cuda")

    def plain(params):
        norm = lambda t, s: t * torch.rsqrt((t ** 2).mean(dim=-1, keepdim=True) + 1e-6) * s  # noqa: E731
        q, k, v = (t.unflatten(-1, (b.heads, b.head_dim)) for t in F.linear(norm(x.double(), params["norm1"]), params["w_qkv"]).chunk(3, dim=-1))
        apart = torch.arange(40, device="cuda")[:, None] - torch.arange(40, device="cuda")[None]
        decay = torch.where(apart >= 0, torch.exp(b.log_decay.double()[:, None, None] * apart.clamp(min=0)), 0.0)
        out = torch.einsum("bhij,bjhd->bihd", torch.einsum("bihd,bjhd->bhij", q, k) * decay, v) * b.head_dim ** -0.5
        h = x.double() + F.linear(out.flatten(2), params["w_out"])
        return h + F.linear(F.silu(F.linear(norm(h, params["norm2"]), params["w_up"], params["b_up"])), params["w_down"])

    params = {n: p.detach().double().requires_grad_() for n, p in b.named_parameters()}
    wants = torch.autograd.grad(((plain(params) - target) ** 2).mean(), list(params.values()))
    loss = ((b(x)[0] - target) ** 2).mean()
    grads = torch.autograd.grad(loss, list(b.parameters()))
    for name, got, want in zip(params, grads, wants):
        assert off(got, want) < 1e-4, name
    # a step against the gradient that should lower the loss by a hundredth of itself, to first order
    length = float(sum((g.double() ** 2).sum() for g in grads))
    with torch.no_grad():
        for p, g in zip(b.parameters(), grads):
            p -= g * (0.01 * float(loss.detach()) / length)
        after = ((b(x)[0] - target) ** 2).mean()
    assert 0.98 * float(loss.detach()) < float(after) < 0.995 * float(loss.detach())


def test_block_in_a_graph():
    """A decoding step of the coded block, captured and replayed on new tokens."""
    c = block(torch.bfloat16, seed=3).coded()
    x = torch.randn(4, 192, device="cuda").bfloat16()
    state = torch.zeros(4, 4, 48, 48, device="cuda")
    c.step(x, state.clone())
    held = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = c.step(held, state)
    state.zero_()
    other = torch.zeros_like(state)
    for seed in range(3):
        torch.manual_seed(seed)
        token = torch.randn(4, 192, device="cuda").bfloat16()
        held.copy_(token)
        graph.replay()
        assert torch.equal(y, c.step(token, other)) and torch.equal(state, other)


def test_no_wait_gave_up():
    import ctypes

    from rx_met_b200 import _cabi
    word = ctypes.c_int(-1)
    assert _cabi.load_library().rxmet_wait_status(ctypes.byref(word)) == 0 and word.value == 0
