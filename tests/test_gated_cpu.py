"""The gated mixer's plain forms agree with one another, and its entry points refuse what needs no GPU to be refused."""
import ctypes as C

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_plain_codes(dtype):
    """No value is off by more than half a step, no smaller step would do, and values survive being kept again."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(6, 100, generator=g) * torch.tensor([1.0, 1e-3, 300.0, 1.0, 0.0, 1.0])[:, None]).to(dtype)
    x[3, 40] = float("inf")
    codes, exponents = gl.keep(x)
    step = torch.exp2(exponents.double()).repeat_interleave(32, dim=1)[:, :100]
    fine = exponents.repeat_interleave(32, dim=1)[:, :100] != 127
    got = gl.values(codes, exponents)
    assert bool(((got - x.double()).abs() <= step / 2)[fine].all()) and torch.isnan(got[3, 32:64]).all() and not torch.isnan(got[3, :32]).any()
    most = codes.abs().int()
    for row in (0, 1, 2, 5):
        for group in range(3):
            assert 64 <= int(most[row, 32 * group:32 * group + 32].max()) <= 127
    again = gl.keep(got[:3].to(dtype))
    assert torch.equal(gl.values(*again), got[:3])


@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
def test_slopes_of_the_plain_activations(activation):
    x = torch.linspace(-9, 9, 301, dtype=torch.float64).requires_grad_()
    value, slope, *_ = gl.curve(x, activation)
    want, = torch.autograd.grad(value.sum(), x)
    assert torch.allclose(slope, want, rtol=1e-12, atol=1e-14)


def test_kept_codes_refuse_what_needs_no_gpu():
    from rx_met_b200 import kept_codes
    x = torch.zeros(4, 32)
    kept = kept_codes.KeptCodes(x.to(torch.int8), torch.zeros(4, 1, dtype=torch.int8), torch.float32)
    for call in (lambda: kept_codes.keep(x), lambda: kept_codes.values(kept), lambda: kept_codes.gated_product(x, x), lambda: kept_codes.weight_gradient(x, kept),
                 lambda: kept_codes.linear(x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="activation"):
        kept_codes.gated_product(x, x, activation="tanh")
    with pytest.raises(RuntimeError, match="type"):
        kept_codes.values(kept._replace(dtype=torch.float64))


class TokenTensor(C.Structure):
    """``rxmet_token_tensor``."""
    _fields_ = [("data", C.c_void_p), ("stride_b", C.c_int64), ("stride_t", C.c_int64)]


class Problem(C.Structure):
    """``rxmet_gated_recurrence``."""
    _fields_ = [(n, C.c_int32) for n in ("batch", "tokens", "width", "type", "tanh_value")] + [(n, TokenTensor) for n in ("forget", "value", "input")] + [("lengths", C.c_void_p)]


def library():
    from rx_met_b200 import _cabi
    lib = _cabi.load_library()
    for name in ("rxmet_gated_recurrence_marks", "rxmet_gated_recurrence_workspace_bytes"):
        getattr(lib, name).restype = C.c_size_t
    return lib


@pytest.mark.parametrize("sizes,message", [((1, 2 ** 30 + 1, 1, 0), b"tokens, at most"), ((2 ** 20, 2 ** 20, 2 ** 20, 1), b"runs of"), ((-1, 1, 1, 0), b"batch -1"), ((1, 1, 0, 0), b"width 0"),
                                           ((1, 1, 1, 3), b"element type"), ((1, 40, 8, 0), b"null pointer")])
def test_the_recurrence_refuses_sizes_that_it_cannot_place(sizes, message):
    lib, none = library(), TokenTensor(None, 1, 1)
    problem = Problem(*sizes, 0, none, none, none, None)
    for call in (lambda: lib.rxmet_gated_recurrence_forward(C.byref(problem), None, None, None, None, None, C.c_size_t(0), None),
                 lambda: lib.rxmet_gated_recurrence_backward(C.byref(problem), None, None, None, None, None, None, None, None, None, C.c_size_t(0), None)):
        assert call() < 0 and message in lib.rxmet_last_error()


@pytest.mark.parametrize("tokens", [33, 64, 1000])
def test_the_recurrence_refuses_the_final_state_of_many_tokens_in_the_place_of_the_state(tokens):
    """A sequence's first tile may still be reading the state when its last one is done."""
    lib, none, some, state = library(), TokenTensor(None, 1, 1), TokenTensor(16, 8 * tokens, 8), C.c_void_p(16)
    problem = Problem(1, tokens, 8, 1, 0, some, some, none, None)
    assert lib.rxmet_gated_recurrence_forward(C.byref(problem), state, C.c_void_p(16), state, None, None, C.c_size_t(0), None) < 0
    assert b"in the place of the state" in lib.rxmet_last_error()


def test_what_the_recurrence_asks_for():
    """Marks of every tile but a sequence's first: 128 tokens of 16 bits, 64 beside an input gate, half of that of floats; a chain's words for tiles that wait for one another."""
    lib, none, some = library(), TokenTensor(None, 1, 1), TokenTensor(16, 1, 1)
    for kind, tile in ((1, 128), (2, 128), (0, 64)):
        for own, gate in ((1, none), (2, some)):
            for tokens in (0, 1, tile // own, tile // own + 1, 1000):
                problem = Problem(3, tokens, 70, kind, 0, none, none, gate, None)
                tiles = max(1, -(-tokens // (tile // own)))
                assert lib.rxmet_gated_recurrence_marks(C.byref(problem)) == 3 * 70 * (tiles - 1)
                groups = -(-tiles // 8)
                words = 3 * 2 * (tiles + groups) * 64 * 8
                assert lib.rxmet_gated_recurrence_workspace_bytes(C.byref(problem)) == (0 if tiles == 1 else -(-(words + 16) // 256) * 256)


def test_kept_codes_refuse_rows_that_they_cannot_place():
    lib = library()
    one, far = C.c_int64(1), C.c_int64(1 << 40)
    calls = [lambda: lib.rxmet_keep_codes(one, 131072, 1, None, one, None, one, None, None), lambda: lib.rxmet_keep_codes(one, 0, 1, None, one, None, one, None, None),
             lambda: lib.rxmet_keep_codes(one, 8, 5, None, one, None, one, None, None), lambda: lib.rxmet_keep_codes(C.c_int64(2), 8, 1, C.c_void_p(16), far, C.c_void_p(16), C.c_int64(16), C.c_void_p(16), None),
             lambda: lib.rxmet_keep_codes(C.c_int64(2), 8, 1, C.c_void_p(16), C.c_int64(8), C.c_void_p(16), C.c_int64(8), C.c_void_p(16), None),
             lambda: lib.rxmet_gated_product(one, 8, 1, 4, C.c_void_p(16), one, C.c_void_p(16), one, C.c_void_p(16), None, None, None, None, one, None),
             lambda: lib.rxmet_kept_weight_gradient(one, 131072, 8, 1, None, one, None, one, None, 0, None, None, C.c_size_t(0), None),
             lambda: lib.rxmet_kept_weight_gradient(far, 8, 8, 1, None, one, None, one, None, 0, None, None, C.c_size_t(0), None)]
    messages = [b"at most 131071", b"of 0 elements", b"element type", b"elements apart", b"16 bytes", b"activation", b"at most", b"at most"]
    for call, message in zip(calls, messages):
        assert call() < 0 and message in lib.rxmet_last_error(), (message, lib.rxmet_last_error())
