"""Where the token mixer's operators can go wrong beside their ordinary inputs: ends of the number range, what is not finite, sizes, memory orders."""
import pytest
import torch

import mixer_lib as ml

pytestmark = pytest.mark.gpu


# ---- rows of codes ------------------------------------------------------------------------------------------------------

def tiny_rows(rows, width, dtype):
    """Rows whose largest magnitudes go down to the smallest number there is, with zeros in them."""
    g = torch.Generator(device="cuda").manual_seed(width)
    x = torch.randn(rows, width, device="cuda", generator=g, dtype=torch.float64)
    tops = torch.tensor([1e-30, 3e-36, 3.8e-37, 3.7e-37, 1e-37, 1e-39, 1e-41, 2.0 ** -149], device="cuda", dtype=torch.float64)
    x = (x / x.abs().amax(dim=1, keepdim=True) * tops[torch.arange(rows, device="cuda") % 8][:, None]).to(dtype)
    x[:, ::3] = 0
    return x


def check_tiny(codes, scale, x):
    most, step, half = x.double().abs().amax(dim=1), scale.double(), 2.0 ** -150   # half: of the smallest number
    ml.within(scale, most / 127, most * 2.0 ** -24 + half)
    # half a step, what the quotient is off by at 127 steps, and what a step that was rounded down leaves of the largest values
    off = (codes.double() * step[:, None] - x.double()).abs()
    assert bool((off <= (step * (0.5 + 127 * 2.0 ** -22) + 127 * half)[:, None]).all())
    assert not codes[x == 0].any() and int(codes.min()) >= -127
    assert bool((codes.abs().amax(dim=1)[most > 1e-38] == 127).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,width", [(8, 64), (8, 50), (3000, 64), (3000, 1000), (2400, 1001), (600, 4096), (8, 16384), (8, 16383)])
def test_codes_of_tiny_rows(rows, width, dtype):
    from rx_met_b200 import rms_norm
    x = tiny_rows(rows, width, dtype)
    check_tiny(*rms_norm.code_rows(x), x)


def test_codes_behind_a_tiny_weight():
    from rx_met_b200 import rms_norm
    x, weight = torch.ones(40, 96, device="cuda"), torch.full((96,), 1e-38, device="cuda")
    weight[::2] = 0
    codes, scale, _ = rms_norm.add_rms_norm_codes(x, weight, eps=0.0)
    check_tiny(codes, scale, weight.expand(40, 96))


# ---- states to the last bits ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [128, 500, 2000])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 48), (40, 128)])
@pytest.mark.parametrize("loud", ["all", "first", "last"])
@pytest.mark.parametrize("small", [1.0, 1e-6])
@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_bits_of_a_state(tokens, Dk, Dv, loud, small, dtype):
    """Relative to the state itself, whichever tokens it comes from.  A chunk's products are added up in 24 steps, each off by 2^-24 of a running sum at most, its operand's terms leave 2^-22 or less: 2^-20.5
    for a sum of independent ones.  Behind it, every chunk multiplies by a power of the decay that is off by 2^-24."""
    from rx_met_b200.decayed_attention import decayed_attention
    g = torch.Generator(device="cuda").manual_seed(2)
    make = lambda d, f: (torch.randn(2, tokens, 4, d, device="cuda", generator=g) * f).to(dtype)  # noqa: E731
    q, k, v, dout = make(Dk, 1.0), make(Dk, 1.0), make(Dv, small), make(Dv, small)
    if loud != "all":   # the tokens that the state, and its gradient, are far from or near to
        quiet = slice(100, None) if loud == "first" else slice(0, max(0, tokens - 100))
        v[:, quiet] = 0
        back = dout.flip(1)
        back[:, quiet] = 0
        dout = back.flip(1)
    decay = torch.tensor([0.0, -0.003, -0.01, -0.03], device="cuda")
    S = torch.zeros(2, 4, Dk, Dv, device="cuda", requires_grad=True)
    out, last = decayed_attention(q, k, v, decay, state=S)
    dstate, = torch.autograd.grad(out, S, dout)
    t = torch.arange(tokens, device="cuda", dtype=torch.float64)
    left, gone = torch.exp(decay.double()[:, None] * (tokens - 1 - t)), torch.exp(decay.double()[:, None] * (t + 1))
    wants = (torch.einsum("bthk,ht,bthv->bhkv", k.double(), left, v.double()), torch.einsum("bthk,ht,bthv->bhkv", q.double(), gone, dout.double()) * Dk ** -0.5)
    for name, got, want in zip(("state", "dstate"), (last.detach(), dstate), wants):
        off = (got.double() - want).flatten(2).norm(dim=2) / want.flatten(2).norm(dim=2)
        assert float(off.max()) < 2.0 ** -20.5 + (tokens // 128) * 2.0 ** -24, (name, off)


@pytest.mark.parametrize("tokens", [128, 500, 2000])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 48), (40, 128)])
@pytest.mark.parametrize("loud", ["all", "first", "last"])
@pytest.mark.parametrize("small", [1.0, 1e-6])
def test_bits_of_a_state_of_half(tokens, Dk, Dv, loud, small):
    """Values of 1e-6 are a few of half's smallest steps: usual gradients without a loss scale."""
    test_bits_of_a_state(tokens, Dk, Dv, loud, small, torch.float16)


# ---- values that are not finite, in front of which nothing may change ------------------------------------------------------------

def attention_problem(tokens, Dk, Dv, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, dout = (torch.randn(2, tokens, h, d, device="cuda", generator=g).to(dtype) for h, d in ((4, Dk), (2, Dk), (2, Dv), (4, Dv)))
    return q, k, v, dout, torch.tensor([0.0, -0.01, -0.3, -3.0], device="cuda")


def apart(got, want, bound, hit):
    """`hit`: what cannot be finite; everything else within its bound."""
    assert not torch.isfinite(got[hit]).any()
    ml.within(got[~hit], want[~hit], bound[~hit])


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (96, 100)])
@pytest.mark.parametrize("tokens,at", [(300, 0), (300, 171), (300, 299), (3000, 2000)])
def test_a_bad_value_reaches_no_earlier_token(tokens, at, Dk, Dv, bad, dtype):
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, _, decay = attention_problem(tokens, Dk, Dv, dtype, seed=1)
    scale = Dk ** -0.5
    want, wanted_last = ml.attend(q, k, v, decay, None, None, scale)
    size, size_last = ml.magnitudes(lambda a, b, c: ml.attend(a, b, c, decay, None, None, scale), (q, k, v))
    bound, bound_last = ml.attention_bound(size, dtype, tokens, Dk, dtype), ml.attention_bound(size_last, torch.float32, tokens, Dk, torch.float32)
    v[0, at, 1, 5] = bad
    out, last = decayed_attention(q, k, v, decay)
    hit, hit_last = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(last, dtype=torch.bool)
    hit[0, at:, 2:, 5] = True
    hit_last[0, 2:, :, 5] = True
    apart(out, want, bound, hit)
    apart(last, wanted_last, bound_last, hit_last)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("of", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("at", [0, 171, 299])
def test_gradients_of_a_bad_value(at, of, dtype):
    """Of a key's or a value's, gradients in front of it do not know; of a query's or an output's, those behind it."""
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, dout, decay = attention_problem(300, 64, 80, dtype, seed=2)
    zero = torch.zeros(2, 4, 64, 80, device="cuda")
    wants = ml.attend_gradients(q, k, v, decay, None, None, 0.125, dout, zero)
    sizes = ml.magnitudes(lambda a, b, c, s, d, e: ml.attend_gradients(a, b, c, decay, s, None, 0.125, d, e), (q, k, v, None, dout, zero))
    dict(q=q, k=k, v=v, dout=dout)[of][0, at, 1, 7] = float("nan")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(decayed_attention(*leaves, decay)[0], leaves, dout)
    dq, dk, dv = (torch.zeros_like(g, dtype=torch.bool) for g in grads)
    query, key = slice(1, 2), slice(0, 1)   # heads of q and dout that read head 0 of k and v: 0 and 1; of its head 1: 2 and 3
    if of == "q":
        dk[0, :at + 1, key, 7] = True
        dv[0, :at + 1, key] = True
    if of == "dout":
        dq[0, at, query] = True
        dk[0, :at + 1, key] = True
        dv[0, :at + 1, key, 7] = True
    if of == "k":
        dq[0, at:, 2:, 7] = True
        dv[0, at, 1] = True
    if of == "v":
        dq[0, at:, 2:] = True
        dk[0, at, 1] = True
    for got, want, size, hit in zip(grads, wants, sizes, (dq, dk, dv)):
        apart(got, want, ml.attention_bound(size, dtype, 300, 80, dtype), hit)


# ---- what torch does with calls -----------------------------------------------------------------------------------------------

def test_calls_are_not_traced():
    """A trace would hold the buffers of the outputs and none of the kernels."""
    from rx_met_b200 import coded_linear, decayed_attention, rms_norm
    x, w = torch.randn(3, 16, device="cuda"), torch.randn(16, device="cuda")
    q, decay, state = torch.randn(3, 5, 1, 16, device="cuda"), -torch.ones(1, device="cuda"), torch.zeros(3, 1, 16, 16, device="cuda")
    codes, scale = rms_norm.code_rows(x)
    for call, inputs in ((lambda a: rms_norm.add_rms_norm(a, w)[0], x), (lambda a: rms_norm.add_rms_norm_codes(a, w)[1], x), (lambda a: rms_norm.code_rows(a)[1], x),
                         (lambda a: coded_linear.coded_linear(codes, a, coded_linear.CodedWeight(codes, scale)), scale),
                         (lambda a: decayed_attention.decayed_attention(a, q, q, decay)[0], q),
                         (lambda a: decayed_attention.decayed_attention_step(a, q[:, 0], q[:, 0], decay, state), q[:, 0].contiguous())):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (inputs,), check_trace=False)
        call(inputs)


def test_second_derivatives_fail():
    """In silence, their terms would be missing from a sum of which others can be differentiated."""
    from rx_met_b200 import rms_norm
    from rx_met_b200.decayed_attention import decayed_attention
    x, r, w = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((3, 16), (3, 16), (16,)))
    q = torch.randn(1, 5, 1, 16, device="cuda", requires_grad=True)
    decay = -torch.ones(1, device="cuda")
    for f, leaves in ((lambda: rms_norm.add_rms_norm(x, w)[0], [x, w]), (lambda: rms_norm.add_rms_norm(x, w, r)[1], [x, r]), (lambda: decayed_attention(q, q, q, decay)[0], [q])):
        first = torch.autograd.grad((f() ** 2).sum(), leaves)
        grads = torch.autograd.grad((f() ** 2).sum(), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, first))
        with pytest.raises(RuntimeError, match="no second derivatives"):
            torch.autograd.grad(sum((g ** 2).sum() for g in grads) + sum((t ** 3).sum() for t in leaves), leaves)


# ---- sizes ------------------------------------------------------------------------------------------------------------------

def test_sizes_of_33_bits_are_refused():
    """They were cut to their lower bits.  Views of one element: nothing of that size is held, and nothing may be copied to it."""
    from rx_met_b200 import rms_norm
    from rx_met_b200.coded_linear import CodedWeight, coded_linear
    from rx_met_b200.decayed_attention import decayed_attention
    more = 2 ** 32
    view = lambda dtype, *shape: torch.ones(1, device="cuda", dtype=dtype).expand(*shape)  # noqa: E731
    of = lambda *shape: view(torch.float32, *shape)  # noqa: E731
    one, small, rows = of(1), of(1, 1, 1, 1), view(torch.int8, 1, more + 64)
    torch.cuda.synchronize()
    held = torch.cuda.max_memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for call in (lambda: rms_norm.add_rms_norm(view(torch.bfloat16, more + 64), view(torch.bfloat16, more + 64)), lambda: rms_norm.code_rows(view(torch.bfloat16, 2, more + 64)),
                 lambda: rms_norm.add_rms_norm_codes(of(1, more + 64), of(more + 64)), lambda: coded_linear(rows, one, CodedWeight(rows, one)),
                 lambda: coded_linear(rows[:, :32], one, CodedWeight(view(torch.int8, more + 3, 32), of(more + 3))),
                 lambda: decayed_attention(*[of(1, more + 2, 1, 1)] * 3, -one), lambda: decayed_attention(*[of(more + 1, 1, 1, 1)] * 3, -one),
                 lambda: decayed_attention(of(1, 1, 1, more + 1), of(1, 1, 1, more + 1), small, -one), lambda: decayed_attention(of(1, 1, more + 1, 1), small, small, -one),
                 lambda: decayed_attention(small, small, of(1, 1, 1, more + 1), -one)):
        with pytest.raises(RuntimeError, match="at most"):
            call()
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() < held + 2 ** 30


# ---- waits that run out -----------------------------------------------------------------------------------------------------------

def test_wait_status_waits_for_all_streams():
    import ctypes as C

    from mixer_abi import library
    side, done, word = torch.cuda.Stream(), torch.cuda.Event(), C.c_int(-1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):   # a stream apart from the legacy one, at work for a fifth of a second
        torch.cuda._sleep(400_000_000)
        done.record()
    assert library().rxmet_wait_status(C.byref(word)) == 0 and word.value == 0
    assert done.query()


def test_no_wait_gave_up():
    import rx_met_b200
    assert rx_met_b200.wait_gave_up() is False


# ---- the C ABI ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("struct", [False, True])
@pytest.mark.parametrize("tokens,Dk,Dv", [(1, 8, 1), (5, 64, 64), (200, 64, 40), (200, 128, 128)])
def test_gradients_of_the_final_state_alone(tokens, Dk, Dv, struct, dtype):
    """No gradient of the outputs: neither the structure nor, in it, the data."""
    import ctypes as C

    from mixer_abi import Heads, Problem, library
    lib = library()
    q, k, v = (torch.randn(2, tokens, h, d, device="cuda").to(dtype) for h, d in ((4, Dk), (2, Dk), (4, Dv)))
    decay, dlast = -torch.rand(4, device="cuda"), torch.randn(2, 4, Dk, Dv, device="cuda")
    problem = Problem(2, tokens, 4, Dk, Dv, ml.TYPES.index(dtype), Heads.of(q), Heads.of(k), Heads.of(v), decay.data_ptr(), None, 0.25)
    grads = [torch.full_like(t, float("nan")) for t in (q, k, v, dlast)]
    size = lib.rxmet_decayed_attention_workspace_bytes(C.byref(problem), 1)
    held = torch.empty(size, dtype=torch.uint8, device="cuda")
    none = C.byref(Heads(None, 0, 0, 0, 4)) if struct else None
    at = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    status = lib.rxmet_decayed_attention_backward(C.byref(problem), None, none, at(dlast), *(at(g) for g in grads), at(held), C.c_size_t(size),
                                                  C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert status == 0, lib.rxmet_last_error()
    zero = torch.zeros(2, tokens, 4, Dv, device="cuda")
    wants = ml.attend_gradients(q, k, v, decay, None, None, 0.25, zero, dlast)
    sizes = ml.magnitudes(lambda a, b, c, s, d, e: ml.attend_gradients(a, b, c, decay, s, None, 0.25, d, e), (q, k, v, None, zero, dlast))
    for got, want, magnitude in zip(grads, wants, sizes):
        # decays of up to e^-200 lead below the normal numbers, where every token's two products may be off by half of the smallest one
        ml.within(got, want, ml.attention_bound(magnitude, dtype, tokens, max(Dk, Dv), got.dtype) + tokens * 2.0 ** -149)


# ---- wide rows of codes -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("rows,width,extra", [(1, 16385, 0), (3, 20000, 8), (700, 28672, 0), (5, 28672, 3), (2, 131071, 0), (0, 20000, 0)])
def test_codes_of_wide_rows(rows, width, extra, dtype):
    """The rows of what goes into a product may be as wide as the product takes them."""
    from rx_met_b200 import rms_norm
    x = torch.randn(rows, width + extra, device="cuda").to(dtype)[:, :width]
    if rows > 1:
        x[1] = 0
    codes, scale = rms_norm.code_rows(x)
    assert codes.shape == (rows, width) and (rows < 2 or (codes.stride(0) % 16 == 0 and scale[1] == 0 and not codes[1].any()))
    if rows:
        assert torch.equal(scale, (x.double().abs().amax(dim=1) / 127).float()) and int(codes.abs().max()) == 127
    step = scale.double()[:, None]
    assert bool(((codes.double() * step - x.double()).abs() <= step * (0.5 + 127 * 2.0 ** -22)).all())


def test_wide_rows_at_the_ends_of_the_range():
    from rx_met_b200 import rms_norm
    x = tiny_rows(8, 20000, torch.float32)
    check_tiny(*rms_norm.code_rows(x), x)
    x[0, 19999], x[1, 0] = float("nan"), float("-inf")
    codes, scale = rms_norm.code_rows(x)
    assert torch.isnan(scale[0]) and torch.isinf(scale[1])
    check_tiny(codes[2:], scale[2:], x[2:])
    with pytest.raises(RuntimeError, match="at most 131071"):
        rms_norm.code_rows(torch.zeros(1, 131072, device="cuda"))
    with pytest.raises(RuntimeError, match="at most 16384"):
        rms_norm.add_rms_norm_codes(torch.zeros(1, 16385, device="cuda"), torch.ones(16385, device="cuda"))


def test_a_block_of_many_hidden_units():
    from rx_met_b200.coded_linear import code_weight, coded_linear
    from rx_met_b200.decay_block import DecayBlock
    from rx_met_b200.rms_norm import code_rows
    torch.manual_seed(0)
    b = DecayBlock(width=64, heads=2, head_dim=32, hidden=20000)
    x = torch.randn(2, 9, 64, device="cuda").bfloat16()
    want = b(x)[0].detach()
    got, _ = b.coded().prefill(x)
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 0.05
    y, w = torch.randn(40, 28672, device="cuda"), torch.randn(24, 28672, device="cuda")
    rows, channels = code_rows(y), code_weight(w)
    out = coded_linear(*rows, channels, dtype=torch.float32)
    exact = (rows[0].double() * rows[1].double()[:, None]) @ (channels.codes.double() * channels.scale.double()[:, None]).T
    assert bool(((out.double() - exact).abs() <= 4 * 2.0 ** -24 * exact.abs() + 1e-30).all())


def test_a_decay_that_could_have_a_gradient():
    """Refused where gradients are recorded, and only there."""
    from rx_met_b200.decayed_attention import decayed_attention, decayed_attention_step
    q, decay = torch.randn(2, 40, 2, 32, device="cuda"), -torch.ones(2, device="cuda")
    leaf, states = decay.clone().requires_grad_(), [torch.zeros(2, 2, 32, 32, device="cuda") for _ in range(2)]
    for call in (lambda: decayed_attention(q, q, q, leaf), lambda: decayed_attention_step(q[:, 0], q[:, 0], q[:, 0], leaf, states[0])):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    with torch.no_grad():
        for a, b in zip(decayed_attention(q, q, q, leaf), decayed_attention(q, q, q, decay)):
            assert torch.equal(a, b)
        steps = [decayed_attention_step(q[:, 0], q[:, 0], q[:, 0], d, s) for d, s in zip((leaf, decay), states)]
    assert torch.equal(*steps) and torch.equal(*states)


# ---- memory orders ------------------------------------------------------------------------------------------------------------

def test_codes_whose_rows_share_memory():
    from rx_met_b200.coded_linear import CodedWeight, coded_linear
    codes, weight = (torch.randint(-127, 128, (n, 96), device="cuda", dtype=torch.int8) for n in (1, 8))
    ones = torch.ones(300, device="cuda")
    windows = torch.randint(-127, 128, (400,), device="cuda", dtype=torch.int8).unfold(0, 96, 1)[:300]
    for rows, channels in ((codes.expand(300, 96), weight), (windows, weight), (windows, codes.expand(8, 96))):
        for inner in (96, 50):
            a, b = rows[:, :inner], channels[:, :inner]
            got = coded_linear(a, ones, CodedWeight(b, ones[:8]), dtype=torch.float32)
            assert torch.equal(got.double(), a.double() @ b.double().T)


# ---- the block ----------------------------------------------------------------------------------------------------------------

def test_a_coded_block_keeps_its_values():
    """Whatever becomes of the block that it was made from."""
    from rx_met_b200.decay_block import DecayBlock
    torch.manual_seed(0)
    b = DecayBlock(width=64, heads=2, head_dim=32, hidden=100)
    c, x = b.coded(), torch.randn(2, 20, 64, device="cuda").bfloat16()
    want = c.prefill(x)
    with torch.no_grad():
        for t in (*b.parameters(), *b.buffers()):
            t.mul_(1.5)
    for got, first in zip(c.prefill(x), want):
        assert torch.equal(got, first)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_block_moved_to_another_type(dtype):
    from rx_met_b200.decay_block import DecayBlock
    torch.manual_seed(0)
    b = DecayBlock(width=64, heads=2, head_dim=32, hidden=100, dtype=torch.float32)
    decay, x = b.log_decay.clone(), torch.randn(2, 20, 64, device="cuda")
    want = b(x)[0].detach().double()
    b = b.cpu().to(dtype).cuda()
    assert b.dtype == dtype and b.log_decay.is_cuda and torch.equal(b.log_decay, decay)
    for got, off in ((b(x.to(dtype))[0], 0.03), (b.coded().prefill(x.to(dtype))[0], 0.05)):
        assert got.dtype == dtype and float((got.detach().double() - want).norm() / want.norm()) < off
    other = DecayBlock(width=64, heads=2, head_dim=32, hidden=100, dtype=dtype)
    other.load_state_dict(b.state_dict())
    assert torch.equal(other(x.to(dtype))[0], b(x.to(dtype))[0])


# ---- what the ordinary tests do not reach -----------------------------------------------------------------------------------------

def apart_rows(t, extra, off):
    """The same rows further apart, `off` elements into memory whose rest is NaN."""
    held = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), device="cuda", dtype=t.dtype)
    held[:, off:off + t.shape[1]] = t
    return held[:, off:off + t.shape[1]]


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("width,extra,off", [(512, 64, 8), (512, 64, 3), (1000, 24, 0), (257, 3, 1), (4096, 8, 8), (7000, 16, 8)])
def test_rows_apart_through_the_ring(width, extra, off, dtype):
    """More rows than the GPU takes at once, with pitches of their own, on 16 bytes and off them; bounds as for rows behind one another."""
    from rx_met_b200 import rms_norm
    from test_rms_norm_gpu import ROUNDINGS
    rows = 3001
    g = torch.Generator(device="cuda").manual_seed(width)
    x, residual, dy, dtotal = (torch.randn(rows, width, device="cuda", generator=g).to(dtype) for _ in range(4))
    weight = 1 + 0.1 * torch.randn(width, device="cuda", generator=g)
    exact = x.double() + residual.double()
    want, _, rms = ml.norm(x, weight, residual, 1e-6)
    want_dx, want_dw = ml.norm_gradients(dy, dtotal, exact, weight, rms)
    d, u = (dy.double() * weight.double()).abs(), (exact * rms).abs()
    size = rms * (d + u * (d * u).mean(dim=1, keepdim=True)) + dtotal.double().abs()
    top = want.abs().amax(dim=1) / 127
    for a, b in ((apart_rows(x, extra, off), apart_rows(residual, extra + 16, off)), (apart_rows(x, extra, off), residual), (x, apart_rows(residual, extra, off))):
        codes, scale, total = rms_norm.add_rms_norm_codes(a, weight, b)
        ml.within(codes.double() * scale.double()[:, None], want, (top * (0.5 + 127 * (3 * ROUNDINGS + 2.0 ** -21)))[:, None].expand_as(want))
        leaves = [a.detach().requires_grad_(), weight.clone().requires_grad_(), b.detach().requires_grad_()]
        y, again = rms_norm.add_rms_norm(*leaves)
        assert torch.equal(again, total)
        ml.within(total, exact, exact.abs() * (ml.UNIT[dtype] + 2.0 ** -23) * 1.01 + ml.TINY[dtype])
        ml.within(y, want, want.abs() * (ml.UNIT[dtype] + ROUNDINGS) * 1.01 + ml.TINY[dtype])
        dx, dweight, dresidual = torch.autograd.grad([y, again], leaves, [dy, dtotal])
        assert torch.equal(dx, dresidual)
        ml.within(dx, want_dx, want_dx.abs() * ml.UNIT[dtype] * 1.01 + size * 3 * ROUNDINGS + ml.TINY[dtype])
        ml.within(dweight, want_dw, (dy.double().abs() * u).sum(dim=0) * (rows / 32 + 64) * 2.0 ** -24)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("rows,inner,outer,activation", [(2500, 1040, 2700, "silu"), (4200, 900, 1300, "gelu"), (600, 2000, 9000, "relu"), (5000, 1040, 1100, "none")])
def test_several_tiles_a_pair(rows, inner, outer, activation, dtype):
    """More tiles than pairs of CTAs, K beyond their ring, ragged edges, all of the epilogue."""
    from test_coded_linear_gpu import check, padded, problem
    codes, scale, weight, weight_scale, bias, residual = problem(rows, inner, outer, seed=rows, dtype=dtype)
    check(padded(codes), scale, padded(weight), weight_scale, bias, activation, residual, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_state", [True, False])
def test_gradients_of_ragged_rows_in_segments(with_state, dtype):
    """Reverse passes whose first segments are empty."""
    from rx_met_b200.decayed_attention import decayed_attention
    g = torch.Generator(device="cuda").manual_seed(3)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q, k, v, dout = (make(4, 3000, h, 64).to(dtype) for h in (2, 1, 2, 2))
    decay, lengths = torch.tensor([-0.002, -0.2], device="cuda"), torch.tensor([3000, 0, 1111, 130], device="cuda")
    S, dlast = (make(4, 2, 64, 64) if with_state else None for _ in range(2))
    leaves = [t.requires_grad_() for t in (q, k, v, S) if t is not None]
    out, last = decayed_attention(q, k, v, decay, state=S, lengths=lengths)
    grads = torch.autograd.grad([out, last] if with_state else [out], leaves, [dout, dlast] if with_state else [dout])
    parts = [None if t is None else t.detach() for t in (q, k, v, S, dout, dlast)]
    wants = ml.attend_gradients(*parts[:3], decay, parts[3], lengths, 0.125, *parts[4:])
    sizes = ml.magnitudes(lambda a, b, c, s, d, e: ml.attend_gradients(a, b, c, decay, s, lengths, 0.125, d, e), parts)
    for got, want, size in zip(grads, wants, sizes):
        ml.within(got, want, ml.attention_bound(size, got.dtype if got.dtype == torch.float32 else dtype, 3000, 64, got.dtype))


def test_a_captured_training_step():
    """With the streams that the gradients' passes run on."""
    from rx_met_b200 import rms_norm
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v = (torch.randn(2, 300, h, 64, device="cuda").bfloat16().requires_grad_() for h in (4, 2, 4))
    decay, w = torch.full((4,), -0.1, device="cuda"), torch.ones(64, device="cuda", requires_grad=True)

    def step():
        out, last = decayed_attention(q, k, rms_norm.add_rms_norm(v, w)[0], decay)
        return [out, last, *torch.autograd.grad([out, last], [q, k, v, w], [torch.ones_like(out), torch.ones_like(last)])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            for t in (q, k, v):
                t.copy_(torch.randn_like(t))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_no_wait_gave_up_in_any_of_these():
    test_no_wait_gave_up()
