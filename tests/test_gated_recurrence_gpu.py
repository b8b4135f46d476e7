"""Gated linear recurrence on the GPU against its formula in 64 bits: sequences, single tokens, gradients, empty rows, odd sizes and strides, refusals."""
import pytest
import torch

import gated_lib as gl
import mixer_lib as ml

pytestmark = pytest.mark.gpu


def tensors(batch, tokens, width, dtype, own=False, seed=0, pad=0):
    """forget, value, input as parts of one projection's result, rows `pad` elements further apart."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    joint = torch.randn(batch, tokens, 3 * width + pad, device="cuda", generator=g) * 1.5
    joint[..., :width] += torch.linspace(0, 6, width, device="cuda")
    joint = joint.to(dtype)
    forget, value, input = (joint[..., i * width:(i + 1) * width] for i in range(3))
    return forget, value, input if own else None


def lengths_of(batch, tokens, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(0, tokens + 1, (batch,), generator=g)
    n[0] = 0
    if batch > 1:
        n[1] = tokens
    return n.cuda()


def underflow(tokens):
    """Below the normal numbers of 32 bits a product is off by up to 2^-150 whatever its size.  A sum that goes through `tokens` of them is off by that for each (gates are at most 1), and of
    the four factors behind it (at most 8 here, together) each adds one more."""
    return 8 * (tokens + 4) * 2.0 ** -150


def check_forward(dtype, got, want):
    out, last = got
    wanted, wanted_last, bound, bound_last = want[:4]
    assert out.dtype == dtype and last.dtype == torch.float32
    ml.within(out, wanted, 1.01 * bound + wanted.abs() * ml.UNIT[dtype] + ml.TINY[dtype] + underflow(out.shape[1]))
    ml.within(last, wanted_last, 1.01 * bound_last + underflow(out.shape[1]))


# fewer tokens than a tile (128), one, one more, several tiles, more tiles than a look back spans (32)
SHAPES = [(1, 1, 1), (3, 1, 100), (2, 2, 64), (2, 16, 31), (1, 17, 65), (3, 127, 64), (2, 128, 96), (2, 129, 2), (3, 300, 130), (2, 1000, 1001), (1, 9000, 40)]


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("batch,tokens,width", SHAPES)
@pytest.mark.parametrize("own,activation", [(False, "none"), (True, "tanh")])
@pytest.mark.parametrize("continued", [False, True])
def test_sequences(batch, tokens, width, own, activation, continued, dtype):
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, input = tensors(batch, tokens, width, dtype, own)
    state = torch.randn(batch, width, device="cuda") if continued else None
    lengths = lengths_of(batch, tokens) if continued else None
    want = gl.recur(forget, value, input, activation, state, lengths)
    check_forward(dtype, gated_recurrence(forget, value, input=input, activation=activation, state=state, lengths=lengths), want)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("batch,tokens,width", SHAPES)
@pytest.mark.parametrize("own,activation", [(False, "none"), (True, "tanh"), (True, "none"), (False, "tanh")])
@pytest.mark.parametrize("continued", [False, True])
def test_gradients(batch, tokens, width, own, activation, continued, dtype):
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, input = tensors(batch, tokens, width, dtype, own, seed=1)
    state = torch.randn(batch, width, device="cuda").requires_grad_() if continued else None
    lengths = lengths_of(batch, tokens) if continued else None
    dout = torch.randn(batch, tokens, width, device="cuda").to(dtype)
    dfinal = torch.randn(batch, width, device="cuda") if continued else None
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (forget, value, input)]
    out, last = gated_recurrence(leaves[0], leaves[1], input=leaves[2], activation=activation, state=state, lengths=lengths)
    wanted = [t for t in (*leaves, state) if t is not None]
    grads = torch.autograd.grad([out, last] if continued else [out], wanted, [dout, dfinal] if continued else [dout])
    detached = None if state is None else state.detach()
    check_forward(dtype, (out.detach(), last.detach()), gl.recur(forget, value, input, activation, detached, lengths))
    wants = gl.recur_gradients(forget, value, input, activation, detached, lengths, dout, dfinal)
    wants = [w for w in (wants if continued else wants[:3]) if w is not None]
    for leaf, grad, (want, bound) in zip(wanted, grads, wants):
        assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
        ml.within(grad, want, 1.01 * bound + want.abs() * ml.UNIT[leaf.dtype] + ml.TINY[leaf.dtype] + underflow(tokens))


def test_gradients_of_single_results():
    """Of the final state alone, of the outputs alone, of some of the inputs: the same numbers as together."""
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, input = (t.detach().requires_grad_() for t in tensors(2, 300, 66, torch.float32, True, seed=2))
    dout, dfinal = torch.randn(2, 300, 66, device="cuda"), torch.randn(2, 66, device="cuda")
    out, last = gated_recurrence(forget, value, input=input)
    only = torch.autograd.grad(last, [forget, value, input], dfinal, retain_graph=True)
    wants = gl.recur_gradients(forget.detach(), value.detach(), input.detach(), "none", None, None, None, dfinal)
    for grad, (want, bound) in zip(only, wants):
        ml.within(grad, want, 1.01 * bound + want.abs() * 2.0 ** -24 + underflow(300))
    together = torch.autograd.grad([out, last], [forget, value, input], [dout, dfinal], retain_graph=True)
    for i, t in enumerate((forget, value, input)):
        alone = torch.autograd.grad([out, last], t, [dout, dfinal], retain_graph=True)[0]
        assert torch.equal(alone, together[i])
    spread = torch.autograd.grad(out.sum(), value)[0]   # a gradient of one number, expanded
    want, bound = gl.recur_gradients(forget.detach(), value.detach(), input.detach(), "none", None, None, torch.ones(2, 300, 66, device="cuda"), None)[1]
    ml.within(spread, want, 1.01 * bound + want.abs() * 2.0 ** -24 + underflow(300))


def test_gradient_against_differences():
    from rx_met_b200.gated_recurrence import gated_recurrence
    leaves = [t.detach().requires_grad_() for t in tensors(2, 40, 9, torch.float32, True, seed=3)] + [torch.randn(2, 9, device="cuda").requires_grad_()]
    a, b = torch.randn(2, 40, 9, device="cuda"), torch.randn(2, 9, device="cuda")

    def loss(forget, value, input, state):
        out, last = gated_recurrence(forget, value, input=input, activation="tanh", state=state)
        return (out.double() * a).sum() + (last.double() * b).sum()

    for i, g in enumerate(torch.autograd.grad(loss(*leaves), leaves)):
        way = torch.randn_like(leaves[i])
        h = 1e-2
        ends = [loss(*[t.detach() + (s * h * way if j == i else 0) for j, t in enumerate(leaves)]) for s in (1, -1)]
        slope, want = float(ends[0] - ends[1]) / (2 * h), float((g.double() * way).sum())
        # third derivative times h^2 / 6, and 738 outputs off by 1e-6 over 2 h
        assert abs(slope - want) <= 2e-3 * max(1.0, float((g.double() * way).abs().sum())), (slope, want)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("batch,width", [(1, 1), (5, 33), (300, 128)])
def test_single_tokens(batch, width, own, dtype):
    from rx_met_b200.gated_recurrence import gated_recurrence_step
    forget, value, input = (None if t is None else t[:, 0] for t in tensors(batch, 1, width, dtype, own, seed=4, pad=3))
    state = torch.randn(batch, width, device="cuda")
    active = torch.arange(batch, device="cuda") % 3 != 1
    one = lambda t: None if t is None else t[:, None]  # noqa: E731
    want = gl.recur(one(forget), one(value), one(input), "tanh", state, active.int())
    new = torch.empty_like(state)
    out = gated_recurrence_step(forget, value, state, input=input, activation="tanh", new_state=new, active=active)
    check_forward(dtype, (out[:, None], new), want)
    kept = state.clone()
    version = state._version
    assert torch.equal(gated_recurrence_step(forget, value, state, input=input, activation="tanh", active=active), out)
    assert torch.equal(state, new) and state._version > version and torch.equal(new[~active], kept[~active])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_prompt_and_its_tokens(dtype):
    from rx_met_b200.gated_recurrence import gated_recurrence, gated_recurrence_step
    forget, value, _ = tensors(3, 200, 70, dtype, seed=5)
    out, last = gated_recurrence(forget, value)
    first, state = gated_recurrence(forget[:, :190], value[:, :190])
    tail = torch.stack([gated_recurrence_step(forget[:, t], value[:, t], state) for t in range(190, 200)], dim=1)
    bound = gl.recur(forget, value)
    ml.within(torch.cat([first, tail], dim=1), out.double(), 2.02 * bound[2] + out.double().abs() * 2.02 * ml.UNIT[dtype] + ml.TINY[dtype])
    ml.within(state, last.double(), 2.02 * bound[3])


def test_strides_alignment_and_reproducibility():
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, input = (t.contiguous() for t in tensors(2, 700, 96, torch.bfloat16, True, seed=6))
    want = gated_recurrence(forget, value, input=input)
    again = gated_recurrence(forget, value, input=input)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    odd = torch.empty(2 * 700 * 96 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 700, 96)      # on 2 bytes
    odd.copy_(forget)
    apart = torch.zeros(2, 700, 96, 2, device="cuda", dtype=torch.bfloat16)
    apart[..., 0] = value                                                                             # elements apart
    four = torch.zeros(2, 700, 98, device="cuda", dtype=torch.bfloat16)[..., 2:]                      # on 4 bytes
    four.copy_(input)
    turned = value.transpose(0, 1).contiguous().transpose(0, 1)                                       # tokens first
    for f, v, i in ((odd, value, input), (forget, apart[..., 0], input), (forget, value, four), (forget, turned, input)):
        got = gated_recurrence(f, v, input=i)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.randn(1, 1, 96, device="cuda").to(torch.bfloat16)
    same = gated_recurrence(wide.expand(2, 700, 96), value, input=input)                             # one gate for all tokens
    assert all(torch.equal(a, b) for a, b in zip(same, gated_recurrence(wide.expand(2, 700, 96).contiguous(), value, input=input)))
    leaves = [t.requires_grad_() for t in (forget, value, input)]
    dout = torch.randn(2, 700, 96, device="cuda").to(torch.bfloat16)
    grads = [torch.autograd.grad(gated_recurrence(forget, value, input=input)[0], leaves, dout) for _ in range(3)]
    assert all(torch.equal(a, b) for g in grads[1:] for a, b in zip(g, grads[0]))


@pytest.mark.parametrize("own,dtype", [(False, torch.bfloat16), (False, torch.float32), (True, torch.float16), (True, torch.float32)])
def test_more_tiles_than_run_at_once(own, dtype):
    """Thousands of tiles, of which every CTA takes several, in sequences of many groups; three times over."""
    from rx_met_b200.gated_recurrence import gated_recurrence
    batch, tokens, width = 8, 3000, 1024
    forget, value, input = (None if t is None else t.detach().requires_grad_() for t in tensors(batch, tokens, width, dtype, own, seed=11))
    dout = torch.randn(batch, tokens, width, device="cuda").to(dtype)
    leaves = [t for t in (forget, value, input) if t is not None]
    results = []
    for _ in range(3):
        out, last = gated_recurrence(forget, value, input=input)
        results.append([out.detach(), last.detach(), *torch.autograd.grad(out, leaves, dout)])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))
    plain = [None if t is None else t.detach() for t in (forget, value, input)]
    check_forward(dtype, results[0][:2], gl.recur(*plain))
    wants = [w for w in gl.recur_gradients(*plain, "none", None, None, dout, None)[:3] if w is not None]
    for grad, (want, bound) in zip(results[0][2:], wants):
        ml.within(grad, want, 1.01 * bound + want.abs() * ml.UNIT[dtype] + ml.TINY[dtype] + underflow(tokens))


def test_calls_side_by_side():
    """Two streams at once, each with a chain of tiles of its own."""
    from rx_met_b200.gated_recurrence import gated_recurrence
    inputs = [tensors(4, 2000, 512, torch.bfloat16, seed=s)[:2] for s in (12, 13)]
    wants = [gated_recurrence(*t) for t in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(5):
        got = []
        for stream, t in zip(streams, inputs):
            with torch.cuda.stream(stream):
                got.append(gated_recurrence(*t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, wants) for a, b in zip(g, w))


def test_empty_ones():
    from rx_met_b200.gated_recurrence import gated_recurrence, gated_recurrence_step
    state = torch.randn(3, 20, device="cuda")
    none = torch.zeros(3, 0, 20, device="cuda").requires_grad_()
    out, last = gated_recurrence(none, none, state=state)
    assert out.shape == (3, 0, 20) and torch.equal(last, state)
    start = state.clone().requires_grad_()
    _, last = gated_recurrence(none, none, state=start)
    assert torch.equal(torch.autograd.grad(last, start, state)[0], state)
    assert not gated_recurrence(none, none)[1].any()
    out, last = gated_recurrence(torch.zeros(0, 5, 20, device="cuda"), torch.zeros(0, 5, 20, device="cuda"))
    assert out.shape == (0, 5, 20) and last.shape == (0, 20)
    assert gated_recurrence_step(torch.zeros(0, 20, device="cuda"), torch.zeros(0, 20, device="cuda"), torch.zeros(0, 20, device="cuda")).shape == (0, 20)


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_what_lies_behind_a_sequence(dtype):
    """Anything there, not finite too, changes nothing, and its gradients are zeros."""
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, input = (t.contiguous() for t in tensors(3, 290, 70, dtype, True, seed=7))
    lengths = torch.tensor([0, 129, 290], device="cuda")
    dout = torch.randn(3, 290, 70, device="cuda").to(dtype)
    results = []
    for bad in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        leaves = []
        for t in (forget, value, input, dout):
            t = t.clone()
            for b in range(3):
                t[b, lengths[b]:] = bad
            leaves.append(t)
        d = leaves.pop()
        leaves = [t.requires_grad_() for t in leaves]
        out, last = gated_recurrence(leaves[0], leaves[1], input=leaves[2], activation="tanh", lengths=lengths)
        grads = torch.autograd.grad([out, last], leaves, [d, torch.ones_like(last)])
        results.append((out, last, *grads))
        for t in (out, *grads):
            assert not t[0].any() and not t[1, 129:].any()
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
    long = gated_recurrence(forget, value, input=input, activation="tanh", lengths=torch.tensor([-5, 129, 2 ** 40], device="cuda"))
    assert torch.equal(long[0], results[0][0]) and torch.equal(long[1], results[0][1])


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_ends_of_the_number_range(dtype):
    """Gates that are shut or open altogether, at both ends of the type."""
    from rx_met_b200.gated_recurrence import gated_recurrence
    most = torch.finfo(dtype).max
    value = torch.randn(1, 200, 6, device="cuda").to(dtype)
    forget = torch.zeros(1, 200, 6, device="cuda", dtype=dtype)
    for d, x in enumerate((most, -most, float("inf"), float("-inf"), 120.0, -120.0)):
        forget[..., d] = x
    state = torch.randn(1, 6, device="cuda")
    out, last = gated_recurrence(forget, value, state=state)
    for d in (0, 2, 4):
        assert torch.equal(last[:, d], state[:, d])
        assert torch.equal(out[:, :, d], state[:, None, d].to(dtype).expand(1, 200))
    for d in (1, 3, 5):
        assert torch.equal(out[:, :, d], value[:, :, d]) and torch.equal(last[:, d], value[:, -1, d].float())


@pytest.mark.parametrize("where", ["forget", "value", "dout"])
def test_a_bad_value_stays_in_its_channel(where):
    from rx_met_b200.gated_recurrence import gated_recurrence
    t = dict(zip(("forget", "value"), tensors(1, 400, 64, torch.float32, seed=8)[:2]), dout=torch.randn(1, 400, 64, device="cuda"))
    t = {n: x.contiguous() for n, x in t.items()}
    clean = gated_recurrence(t["forget"], t["value"])[0]
    t[where][0, 200, 5] = float("nan")
    leaves = [t["forget"].requires_grad_(), t["value"].requires_grad_()]
    out, last = gated_recurrence(*leaves)
    grads = torch.autograd.grad(out, leaves, t["dout"])
    others = torch.arange(64, device="cuda") != 5
    assert all(bool(torch.isfinite(g[..., others]).all()) for g in (out, *grads))
    if where == "dout":
        assert torch.equal(out, clean) and bool(torch.isnan(grads[1][0, :201, 5]).all()) and bool(torch.isfinite(grads[1][0, 201:, 5]).all())
    else:
        assert torch.equal(out[:, :200], clean[:, :200]) and bool(torch.isnan(out[0, 200:, 5]).all()) and bool(torch.isnan(last[0, 5]))


def test_graphs_streams_and_traces():
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, _ = (t if t is None else t.contiguous() for t in tensors(2, 600, 80, torch.bfloat16, seed=9))
    want = gated_recurrence(forget, value)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gated_recurrence(forget, value)
        for _ in range(2):
            gated_recurrence(forget, value)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    x, y = torch.zeros_like(forget), torch.zeros_like(value)
    with torch.cuda.graph(graph):
        held = gated_recurrence(x, y)
    x.copy_(forget)
    y.copy_(value)
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda a: gated_recurrence(a, value)[0], forget)
    leaf = forget.clone().requires_grad_()
    first = torch.autograd.grad(gated_recurrence(leaf, value)[0].float().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(first.float().sum(), leaf)


def test_a_captured_training_step():
    from rx_met_b200.gated_recurrence import gated_recurrence
    forget, value, _ = tensors(2, 300, 40, torch.float16, seed=10)
    dout = torch.randn(2, 300, 40, device="cuda").half()
    leaves = [forget.contiguous().clone().requires_grad_(), value.contiguous().clone().requires_grad_()]
    want = torch.autograd.grad(gated_recurrence(*leaves)[0], leaves, dout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(gated_recurrence(*leaves)[0], leaves, dout)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_as_many_rows_as_there_can_be():
    """One more row than a batch may have does not fit into 32 bits, and the last block has threads for it."""
    from rx_met_b200.gated_recurrence import gated_recurrence_step
    rows = 2 ** 31 - 1
    forget, value = torch.zeros(rows, 1, device="cuda", dtype=torch.float16), torch.ones(rows, 1, device="cuda", dtype=torch.float16)
    state = torch.zeros(rows, 1, device="cuda")
    out = gated_recurrence_step(forget, value, state)
    assert all(t.amin().item() == 0.5 and t.amax().item() == 0.5 for t in (out, state))   # h = 0 / 2 + 1 / 2
    del forget, value, state, out
    torch.cuda.empty_cache()


def test_refusals():
    from rx_met_b200.gated_recurrence import gated_recurrence, gated_recurrence_step
    x = torch.zeros(2, 8, 16, device="cuda", dtype=torch.bfloat16)
    state = torch.zeros(2, 16, device="cuda")
    for call in (lambda: gated_recurrence(x, x[:, :7]), lambda: gated_recurrence(x, x.half()), lambda: gated_recurrence(x.double(), x.double()),
                 lambda: gated_recurrence(x, x, input=x[:1]), lambda: gated_recurrence(x, x, state=state[:1]), lambda: gated_recurrence(x, x, state=state.half()),
                 lambda: gated_recurrence(x, x, lengths=torch.zeros(3, device="cuda", dtype=torch.int32)), lambda: gated_recurrence(x, x, lengths=torch.zeros(2, device="cuda")),
                 lambda: gated_recurrence(x, x.cpu()), lambda: gated_recurrence(x, x, lengths=torch.zeros(2, dtype=torch.int32)), lambda: gated_recurrence(x[..., :0], x[..., :0]),
                 lambda: gated_recurrence(x[0], x[0]), lambda: gated_recurrence_step(x, x, state), lambda: gated_recurrence_step(x[:, 0], x[:, 0], state, new_state=state.t().contiguous().t()),
                 lambda: gated_recurrence_step(x[:, 0].float().requires_grad_(), x[:, 0].float(), state)):
        with pytest.raises(RuntimeError):
            call()
    held = torch.zeros(3, 16, device="cuda")
    with pytest.raises(RuntimeError, match="overlap|memory"):
        gated_recurrence_step(x[:, 0], x[:, 0], held[:2], new_state=held[1:])
