"""Linear attention with decays on the GPU against its recurrence in 64 bits: lengths, states, shared heads, strides, gradients, refusals."""
import math

import pytest
import torch

import mixer_lib as ml

pytestmark = pytest.mark.gpu


def problem(B, T, H, Hk, Dk, Dv, dtype, seed=0, state=False, joint=True, Hq=None, Hv=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    Hq, Hv = Hq or H, Hv or Hk
    if joint:   # views of one projection's result
        held = torch.randn(B, T, Hq * Dk + Hk * Dk + Hv * Dv, device="cuda", generator=g).to(dtype)
        q, k, v = held.split([Hq * Dk, Hk * Dk, Hv * Dv], dim=-1)
        q, k, v = q.view(B, T, Hq, Dk), k.view(B, T, Hk, Dk), v.view(B, T, Hv, Dv)
    else:
        q, k, v = (torch.randn(B, T, h, d, device="cuda", generator=g).to(dtype) for h, d in ((Hq, Dk), (Hk, Dk), (Hv, Dv)))
    decay = torch.log1p(-torch.exp2(-torch.linspace(0.5, 9, H, device="cuda")))
    S = torch.randn(B, H, Dk, Dv, device="cuda", generator=g) if state else None
    return q, k, v, decay, S


def check_forward(q, k, v, decay, state, lengths, scale=None):
    from rx_met_b200.decayed_attention import decayed_attention
    out, last = decayed_attention(q, k, v, decay, state=state, lengths=lengths, scale=scale)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, wanted_last = ml.attend(q, k, v, decay, state, lengths, scale)
    size, size_last = ml.magnitudes(lambda a, b, c, s: ml.attend(a, b, c, decay, s, lengths, abs(scale)), (q, k, v, state))
    tokens, dim = q.shape[1], q.shape[3]
    assert out.dtype == q.dtype and last.dtype == torch.float32
    ml.within(out, want, ml.attention_bound(size, q.dtype, tokens, dim, q.dtype))
    ml.within(last, wanted_last, ml.attention_bound(size_last, torch.float32, tokens, dim, torch.float32))
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            assert not out[b, max(n, 0):].any()
    return out, last


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 64, 127, 128, 129, 300])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 128), (40, 72)])
def test_lengths_of_sequences(tokens, Dk, Dv, dtype):
    check_forward(*problem(2, tokens, 4, 4, Dk, Dv, dtype, seed=tokens, state=tokens % 2 == 0), None)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 1), (8, 8), (16, 128), (128, 16), (33, 50), (96, 64), (128, 7), (100, 100), (80, 120)])
@pytest.mark.parametrize("state", [False, True])
def test_head_sizes(Dk, Dv, state, dtype):
    check_forward(*problem(2, 150, 2, 2, Dk, Dv, dtype, seed=Dk, state=state), None)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("H,Hq,Hk,Hv", [(4, 4, 1, 1), (6, 6, 2, 3), (4, 1, 1, 4), (8, 8, 8, 2)])
def test_shared_heads(H, Hq, Hk, Hv, dtype):
    check_forward(*problem(2, 140, H, Hk, 64, 32, dtype, seed=H, state=True, Hq=Hq, Hv=Hv), None)


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("tokens", [1, 50, 400])
@pytest.mark.parametrize("index_type", [torch.int32, torch.int64])
def test_ragged_rows(tokens, index_type, dtype):
    """Rows of no tokens, of all, more than there are and fewer than none; what lies behind a row's end holds NaN and infinities."""
    q, k, v, decay, state = problem(6, tokens, 4, 2, 64, 64, dtype, seed=5, state=True, joint=False)
    lengths = torch.tensor([0, tokens, tokens // 2, tokens + 7, -3, max(tokens - 1, 0)], device="cuda", dtype=index_type)
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v):
            t[b, max(n, 0):] = float("nan") if b % 2 else float("inf")
    _, last = check_forward(q, k, v, decay, state, lengths)
    assert torch.equal(last[[0, 4]], state[[0, 4]])


def test_lengths_beyond_32_bits():
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, decay, state = problem(2, 40, 2, 2, 32, 32, torch.bfloat16, seed=3, state=True)
    want = decayed_attention(q, k, v, decay, state=state, lengths=torch.tensor([40, 0], device="cuda"))
    got = decayed_attention(q, k, v, decay, state=state, lengths=torch.tensor([2 ** 32 + 1, -2 ** 40], device="cuda"))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("queries,keys,values", [(1.0, 1e-4, 1.0), (1.0, 1.0, 1e-4), (1e-4, 300.0, 300.0)])
def test_small_and_large_values(queries, keys, values, dtype):
    """Scores and states near both ends of half's range: the bounds hold relative to the magnitudes."""
    q, k, v, decay, state = problem(2, 300, 2, 2, 64, 64, dtype, seed=13, state=True)
    q, k, v, state = ((t.double() * f).to(t.dtype) for t, f in ((q, queries), (k, keys), (v, values), (state, keys * values)))
    from rx_met_b200.decayed_attention import decayed_attention
    out, last = decayed_attention(q, k, v, decay, state=state)
    want, wanted_last = ml.attend(q, k, v, decay, state, None, 0.125)
    magnitude, magnitude_last = ml.magnitudes(lambda a, b, c, s: ml.attend(a, b, c, decay, s, None, 0.125), (q, k, v, state))
    assert want.abs().max() < torch.finfo(dtype).max
    # operands are scaled to the top of half's range, so that what they lose is relative to a row's largest: as much as its unit once more
    bound = ml.attention_bound(magnitude, dtype, 300, 64, dtype) - (192 * 2.0 ** -25 * 5 if dtype == torch.float16 else 0)
    ml.within(out, want, bound + magnitude * ml.UNIT[dtype])
    ml.within(last, wanted_last, ml.attention_bound(magnitude_last, torch.float32, 300, 64, torch.float32))


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("tokens", [5, 300])
def test_decays(tokens, dtype):
    """No decay, hardly any memory, none at all."""
    q, k, v, _, state = problem(2, tokens, 5, 5, 64, 64, dtype, seed=6, state=True)
    check_forward(q, k, v, torch.tensor([0.0, -1e-4, -5.0, -90.0, -math.inf], device="cuda"), state, None)


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_long_sequences_of_few_heads(dtype):
    q, k, v, decay, state = problem(1, 3001, 2, 1, 64, 64, dtype, seed=7, state=True)
    check_forward(q, k, v, decay, state, None, scale=-0.3)
    check_forward(q, k, v, decay, None, torch.tensor([2222], device="cuda"))


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_in_parts_and_by_tokens(dtype):
    """A sequence in two calls, and its last tokens one by one, out of place and in place."""
    from rx_met_b200.decayed_attention import decayed_attention, decayed_attention_step
    q, k, v, decay, _ = problem(3, 210, 4, 2, 64, 40, dtype, seed=8)
    whole, last = decayed_attention(q, k, v, decay)
    want, wanted_last = ml.attend(q, k, v, decay, None, None, 0.125)
    size, size_last = ml.magnitudes(lambda a, b, c: ml.attend(a, b, c, decay, None, None, 0.125), (q, k, v))
    first, state = decayed_attention(q[:, :200], k[:, :200], v[:, :200], decay)
    parts = [first]
    for t in range(200, 210):
        if t % 2:
            parts.append(decayed_attention_step(q[:, t], k[:, t], v[:, t], decay, state)[:, None])
        else:
            new = torch.full_like(state, float("nan"))
            before = state.clone()
            parts.append(decayed_attention_step(q[:, t], k[:, t], v[:, t], decay, state, new_state=new)[:, None])
            assert torch.equal(state, before)
            state = new
    ml.within(torch.cat(parts, dim=1), want, ml.attention_bound(size, dtype, 210, 64, dtype))
    ml.within(state, wanted_last, ml.attention_bound(size_last, torch.float32, 210, 64, torch.float32))
    active = torch.tensor([True, False, True], device="cuda")
    before = state.clone()
    out = decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state, active=active)
    assert torch.equal(state[1], before[1]) and not out[1].any() and not torch.equal(state[0], before[0])


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv,state,ragged", [(1, 1, 1, 1, 8, 8, True, False), (2, 33, 2, 2, 40, 72, True, False), (2, 128, 4, 4, 64, 64, False, False),
                                                         (3, 300, 4, 1, 96, 64, True, True), (2, 257, 2, 2, 128, 128, False, True), (2, 200, 4, 2, 33, 50, True, True),
                                                         (1, 2000, 2, 2, 64, 64, True, False)])
def test_gradients(B, T, H, Hk, Dk, Dv, state, ragged, dtype):
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, decay, S = problem(B, T, H, Hk, Dk, Dv, dtype, seed=T, state=state)
    lengths = torch.tensor([T, 0, T // 2][:B], device="cuda") if ragged else None
    dout = torch.randn(B, T, H, Dv, device="cuda").to(dtype)
    dlast = torch.randn(B, H, Dk, Dv, device="cuda") if state else None
    leaves = [t.detach().requires_grad_() for t in ((q, k, v, S) if state else (q, k, v))]
    out, last = decayed_attention(*leaves[:3], decay, state=leaves[3] if state else None, lengths=lengths)
    grads = torch.autograd.grad([out, last] if state else [out], leaves, [dout, dlast] if state else [dout])
    scale = Dk ** -0.5
    wants = ml.attend_gradients(q, k, v, decay, S, lengths, scale, dout, dlast)
    sizes = ml.magnitudes(lambda a, b, c, s, d, e: ml.attend_gradients(a, b, c, decay, s, lengths, scale, d, e), (q, k, v, S, dout, dlast))
    for name, got, want, size, kind in zip(("dq", "dk", "dv", "dstate"), grads, wants, sizes, (dtype, dtype, dtype, torch.float32)):
        assert got.dtype == kind, name
        ml.within(got, want, ml.attention_bound(size, torch.float32 if name == "dstate" else dtype, T, max(Dk, Dv), kind))


def test_gradient_against_differences():
    """The operator is linear in each of q, k, v and state, so that a central difference has no error but its roundings."""
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, decay, state = problem(2, 70, 4, 2, 24, 40, torch.float32, seed=11, state=True)
    lengths = torch.tensor([70, 31], device="cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, state)]
    a, b = torch.randn(2, 70, 4, 40, device="cuda"), torch.randn(2, 4, 24, 40, device="cuda")

    def loss(q, k, v, s):
        out, last = decayed_attention(q, k, v, decay, state=s, lengths=lengths)
        return (out.double() * a).sum() + (last.double() * b).sum()

    for i, g in enumerate(torch.autograd.grad(loss(*leaves), leaves)):
        way = torch.randn_like(leaves[i])
        ends = [loss(*[t.detach() + (s * way if j == i else 0) for j, t in enumerate(leaves)]) for s in (1, -1)]
        slope, want = float(ends[0] - ends[1]) / 2, float((g.double() * way).sum())
        size = float((g.double() * way).abs().sum()) + abs(float(ends[0])) + abs(float(ends[1]))
        assert abs(slope - want) <= 1e-4 * size, (i, slope, want)


def test_strides_streams_and_reproducibility():
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, decay, state = problem(3, 200, 4, 4, 64, 64, torch.bfloat16, seed=12, state=True, joint=False)
    base = decayed_attention(q, k, v, decay, state=state)
    time_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    elements_apart = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    off_grid = []
    for t in (q, k, v):
        held = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        held.copy_(t)
        off_grid.append(held)
    one_row = [t[:1].expand(3, -1, -1, -1) for t in (q, k, v)]   # a stride of zero
    for views in (time_major, heads_first, elements_apart, off_grid):
        got = decayed_attention(*views, decay, state=state.transpose(2, 3).contiguous().transpose(2, 3))
        size, _ = ml.magnitudes(lambda a, b, c, s: ml.attend(a, b, c, decay, s, None, 0.125), (q, k, v, state))
        ml.within(got[0], base[0].double(), 2 * ml.attention_bound(size, torch.bfloat16, 200, 64, torch.bfloat16))
    got = decayed_attention(*one_row, decay, state=state[:1].expand(3, -1, -1, -1))
    assert torch.equal(got[0][0], base[0][0]) and torch.equal(got[0][2], base[0][0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = decayed_attention(q, k, v, decay, state=state)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], base[0]) and torch.equal(other[1], base[1])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    runs = [torch.autograd.grad(decayed_attention(*leaves, decay)[0], leaves, torch.ones_like(base[0])) for _ in range(3)]
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))
    broadcast = torch.autograd.grad(decayed_attention(*leaves, decay)[0].sum(), leaves)   # a gradient of strides zero
    assert all(torch.equal(a, b) for a, b in zip(broadcast, runs[0]))
    only_state = torch.autograd.grad(decayed_attention(*leaves, decay)[1].sum(), leaves[1:])
    assert all(torch.isfinite(g).all() for g in only_state)


def test_gradients_in_a_thread_without_a_context():
    """The autograd engine's thread may not have touched the device before."""
    import subprocess
    import sys
    from pathlib import Path
    code = ("import torch; from rx_met_b200.decayed_attention import decayed_attention\n"
            "q, k, v = (torch.randn(2, 256, 2, 64, device='cuda', dtype=torch.bfloat16, requires_grad=True) for _ in range(3))\n"
            "decay = -torch.ones(2, device='cuda')\n"
            "warm = torch.empty(1 << 22, device='cuda'); del warm\n"
            "out, _ = decayed_attention(q, k, v, decay)\n"
            "grads = torch.autograd.grad([out], [q, k, v], [torch.ones_like(out)])\n"
            "assert all(torch.isfinite(g).all() for g in grads)\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_nothing_to_do():
    from rx_met_b200.decayed_attention import decayed_attention
    q, k, v, decay, state = problem(2, 0, 2, 2, 16, 16, torch.bfloat16, state=True, joint=False)
    out, last = decayed_attention(q, k, v, decay, state=state)
    assert out.shape == (2, 0, 2, 16) and torch.equal(last, state)
    out, last = decayed_attention(q, k, v, decay)
    assert not last.any()
    q, k, v, decay, state = problem(0, 5, 2, 2, 16, 16, torch.bfloat16, state=True, joint=False)
    out, last = decayed_attention(q, k, v, decay, state=state)
    assert out.shape == (0, 5, 2, 16) and last.shape == (0, 2, 16, 16)


def test_a_captured_step_replays():
    from rx_met_b200.decayed_attention import decayed_attention, decayed_attention_step
    q, k, v, decay, state = problem(2, 300, 2, 2, 64, 64, torch.bfloat16, state=True)
    want = decayed_attention(q, k, v, decay, state=state)
    kept = state.clone()
    decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, kept.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = decayed_attention(q, k, v, decay, state=state)
        step = decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, kept)
    kept.copy_(state)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    again = state.clone()
    assert torch.equal(step, decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, again)) and torch.equal(again, kept)


def test_refusals():
    from rx_met_b200.decayed_attention import decayed_attention, decayed_attention_step
    q, k, v, decay, state = problem(2, 5, 4, 2, 16, 24, torch.bfloat16, state=True)
    bad = [dict(q=q.cpu()), dict(k=k.half()), dict(v=v[:, :4]), dict(k=k[..., :8]), dict(q=q[:, 0]), dict(log_decay=decay[:3]), dict(log_decay=decay.double()),
           dict(log_decay=decay.clone().requires_grad_()), dict(state=state[..., :8]), dict(state=state.half()), dict(lengths=torch.ones(3, device="cuda", dtype=torch.int32)),
           dict(lengths=torch.ones(2, device="cuda")), dict(lengths=torch.ones(2, dtype=torch.int32)), dict(q=q.double(), k=k.double(), v=v.double()),
           dict(q=torch.zeros(2, 5, 4, 136, device="cuda", dtype=torch.bfloat16), k=torch.zeros(2, 5, 4, 136, device="cuda", dtype=torch.bfloat16), state=None)]
    for change in bad:
        arguments = dict(dict(q=q, k=k, v=v, log_decay=decay, state=state), **change)
        with pytest.raises(RuntimeError):
            decayed_attention(**arguments)
    for scale in (0.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            decayed_attention(q, k, v, decay, scale=scale)
    with pytest.raises(RuntimeError):
        decayed_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state, new_state=state.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(RuntimeError):
        decayed_attention_step(q[:, 0].detach().requires_grad_(), k[:, 0], v[:, 0], decay, state)
