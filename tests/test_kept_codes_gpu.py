"""Activations kept in 8 bits on the GPU against their formulas in 64 bits: codes, values, the gated product, gradients of weights, a layer; odd sizes and strides, refusals."""
import pytest
import torch

import gated_lib as gl
import mixer_lib as ml

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (3, 7), (2, 32), (5, 33), (1, 1024), (9, 1001), (300, 264), (777, 512), (64, 8192), (3, 131071)]


def rows(count, width, dtype, seed=0, pitch=None):
    """Groups of sizes from 2^-30 to 2^10, with zeros, ties and whole numbers of steps among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(count, pitch or width, device="cuda", generator=g, dtype=torch.float64)
    scale = torch.exp2(torch.randint(-30, 10, (count, -(-x.shape[1] // 32)), device="cuda", generator=g).double())
    x = x * scale.repeat_interleave(32, dim=1)[:, :x.shape[1]]
    x = x.to(dtype)
    if width >= 64:
        x[0, 32:64] = 0
    if width >= 32:
        x[-1, :32] = torch.arange(-16, 16, device="cuda") + 0.5
        x[-1, 0] = 127
    return x[:, :width]


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("count,width", SHAPES)
def test_codes_and_values(count, width, dtype):
    from rx_met_b200 import kept_codes
    x = rows(count, width, dtype)
    kept = kept_codes.keep(x)
    codes, exponents = gl.keep(x)
    assert kept.dtype == dtype and torch.equal(kept.exponents, exponents) and torch.equal(kept.codes, codes)
    assert kept.codes.stride(0) % 16 == 0 or count == 1
    got = kept_codes.values(kept)
    assert got.dtype == dtype and torch.equal(got.double(), gl.values(codes, exponents))


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_codes_at_the_ends_of_the_number_range(dtype):
    from rx_met_b200 import kept_codes
    info = torch.finfo(dtype)
    tops = [info.max, info.tiny, info.smallest_normal, 127.0, 127.5, 1.984375, 1.9921875, 63.5, 0.0, float("inf"), float("nan"), -float("inf"), 1e-7]
    x = torch.zeros(len(tops), 64, device="cuda", dtype=dtype)
    for i, top in enumerate(tops):
        x[i, 40] = top
        x[i, 41] = -top / 3
        x[i, 3] = 1.0
    x[:, 10] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps   # the smallest number there is
    kept = kept_codes.keep(x)
    codes, exponents = gl.keep(x)
    assert torch.equal(kept.exponents, exponents) and torch.equal(kept.codes, codes)
    assert bool((exponents[9:12, 1] == 127).all())
    got, want = kept_codes.values(kept), gl.values(codes, exponents)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.double().nan_to_num(7.0), want.to(dtype).double().nan_to_num(7.0))


def test_codes_of_strides_and_shapes():
    from rx_met_b200 import kept_codes
    x = rows(40, 256, torch.bfloat16, pitch=300)
    want = kept_codes.keep(x.contiguous())
    odd = torch.empty(40 * 256 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(40, 256)
    odd.copy_(x)
    for y in (x, odd, x.t().contiguous().t()):
        got = kept_codes.keep(y)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.exponents, want.exponents)
    deep = kept_codes.keep(x.contiguous().view(5, 8, 256))
    assert deep.codes.shape == (5, 8, 256) and deep.exponents.shape == (5, 8, 8) and torch.equal(deep.codes.view(40, 256), want.codes)
    assert kept_codes.values(deep).shape == (5, 8, 256)
    line = kept_codes.keep(x[0, :50].contiguous())
    assert line.codes.shape == (50,) and line.exponents.shape == (2,)
    # codes that a caller laid out another way are copied
    loose = kept_codes.KeptCodes(torch.cat([want.codes, want.codes[:, :3]], dim=1)[:, :256], want.exponents.t().contiguous().t(), want.dtype)
    assert torch.equal(kept_codes.values(loose), kept_codes.values(want))
    same = kept_codes.KeptCodes(want.codes[:1].expand(40, 256), want.exponents[:1].expand(40, 8), want.dtype)
    assert torch.equal(kept_codes.values(same), kept_codes.values(want)[:1].expand(40, 256))
    none = kept_codes.keep(x[:0])
    assert none.codes.shape == (0, 256) and kept_codes.values(none).shape == (0, 256)
    held = torch.randn(4, 64, device="cuda").requires_grad_()
    assert not kept_codes.values(kept_codes.keep(held)).requires_grad


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("count,width", SHAPES[:-1])
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
def test_gated_product(count, width, activation, dtype):
    from rx_met_b200 import kept_codes
    g = torch.Generator(device="cuda").manual_seed(3)
    joint = (torch.randn(count, 2 * width, device="cuda", generator=g) * 3).to(dtype)
    gate, up = (t.detach().requires_grad_() for t in joint.split(width, dim=1))
    dy = torch.randn(count, width, device="cuda", generator=g).to(dtype)
    y = kept_codes.gated_product(gate, up, activation=activation)
    dgate, dup = torch.autograd.grad(y, [gate, up], dy)
    assert y.dtype == dgate.dtype == dup.dtype == dtype
    value, _, off, _ = gl.curve(gate.detach().double(), activation)
    # below the normal numbers of 32 bits a curve is off by up to six of the smallest steps, 2^-149, whatever its size, and so is each product behind it; times factors of at
    # most 16 each, 5 standard deviations of 3: 2^11 covers 8 * 16^2
    unit, tiny, rounding = ml.UNIT[dtype], ml.TINY[dtype] + 2.0 ** (11 - 149), 2.0 ** -23
    other = up.detach().double()
    ml.within(y.detach(), value * other, (value * other).abs() * (unit + rounding) * 1.01 + off * other.abs() * 1.01 + tiny)
    kept_gate, kept_up = (gl.values(*gl.keep(t.detach())) for t in (gate, up))
    value, slope, off, slope_off = gl.curve(kept_gate, activation)
    d = dy.double()
    want = d * kept_up * slope
    ml.within(dgate, want, want.abs() * (unit + 2 * rounding) * 1.01 + (d * kept_up).abs() * slope_off * 1.01 + tiny)
    ml.within(dup, d * value, (d * value).abs() * (unit + rounding) * 1.01 + d.abs() * off * 1.01 + tiny)
    with torch.no_grad():
        assert torch.equal(kept_codes.gated_product(gate, up, activation=activation), y)


def test_gated_product_of_one_gradient_and_of_strides():
    from rx_met_b200 import kept_codes
    gate, up = rows(40, 96, torch.float32, seed=4), rows(40, 96, torch.float32, seed=5, pitch=101)
    dy = torch.randn(40, 96, device="cuda")
    leaves = [gate.clone().requires_grad_(), up.clone().requires_grad_()]
    want = torch.autograd.grad(kept_codes.gated_product(*leaves), leaves, dy)
    for i in range(2):
        args = [leaves[j] if i == j else leaves[j].detach() for j in range(2)]
        assert torch.equal(torch.autograd.grad(kept_codes.gated_product(*args), leaves[i], dy)[0], want[i])
    deep = [t.detach().view(4, 10, 96).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_() for t in leaves]
    y = kept_codes.gated_product(*deep)
    got = torch.autograd.grad(y, deep, dy.view(4, 10, 96).expand(4, 10, 96))
    assert y.shape == (4, 10, 96) and all(torch.equal(a.view(40, 96), b) for a, b in zip(got, want))
    spread = torch.autograd.grad(kept_codes.gated_product(*leaves).sum(), leaves[1])[0]
    assert torch.equal(spread, torch.autograd.grad(kept_codes.gated_product(*leaves), leaves[1], torch.ones_like(dy))[0])
    none = leaves[0][:0]
    assert kept_codes.gated_product(none, none).shape == (0, 96)
    first = torch.autograd.grad(kept_codes.gated_product(*leaves), leaves, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first[0].sum(), leaves[1])


def test_gated_product_against_differences():
    """At values that codes hold exactly, the gradient is that of the product itself."""
    from rx_met_b200 import kept_codes
    for activation in ("silu", "gelu", "none"):
        leaves = [kept_codes.values(kept_codes.keep(torch.randn(6, 70, device="cuda"))).requires_grad_() for _ in range(2)]
        a = torch.randn(6, 70, device="cuda")
        loss = lambda g, u: (kept_codes.gated_product(g, u, activation=activation).double() * a).sum()  # noqa: E731
        for i, grad in enumerate(torch.autograd.grad(loss(*leaves), leaves)):
            way, h = torch.randn(6, 70, device="cuda"), 1e-2
            ends = [loss(*[t.detach() + (s * h * way if j == i else 0) for j, t in enumerate(leaves)]) for s in (1, -1)]
            slope, want = float(ends[0] - ends[1]) / (2 * h), float((grad.double() * way).sum())
            # third derivative times h^2 / 6, and 420 outputs off by 1e-6 over 2 h
            assert abs(slope - want) <= 2e-3 * max(1.0, float((grad.double() * way).abs().sum()))


def weight_bound(dy, value, tokens):
    """Products are exact.  A step of the tensor cores adds sixteen of them to a running sum and cuts each addend to the sum's last place, 2^-23 of a magnitude for every step; then the parts, up to 74."""
    return dy.double().abs().T @ value.abs() * (tokens / 16 + 17 + 74) * 2.0 ** -23


WEIGHTS = [(1, 1, 1), (1, 40, 8), (7, 33, 5), (64, 64, 64), (65, 128, 256), (200, 300, 264), (130, 777, 1100), (1000, 512, 96), (3000, 257, 513), (5000, 64, 2048), (700, 2048, 64)]


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("tokens,inner,outer", WEIGHTS)
def test_weight_gradient(tokens, inner, outer, dtype):
    from rx_met_b200 import kept_codes
    g = torch.Generator(device="cuda").manual_seed(6)
    x = (torch.randn(tokens, inner, device="cuda", generator=g) * torch.exp2(torch.randint(-4, 4, (tokens, 1), device="cuda", generator=g))).to(dtype)
    dy = torch.randn(tokens, outer, device="cuda", generator=g).to(dtype)
    kept = kept_codes.keep(x)
    value = gl.values(*gl.keep(x))
    want, bound = dy.double().T @ value, weight_bound(dy, value, tokens)
    for out in (dtype, torch.float32):
        got = kept_codes.weight_gradient(dy, kept, dtype=out)
        assert got.dtype == out
        ml.within(got, want, bound + (want.abs() + bound) * ml.UNIT[out] + ml.TINY[out])
    assert torch.equal(kept_codes.weight_gradient(dy, kept), kept_codes.weight_gradient(dy, kept, dtype=dtype))


def test_weight_gradient_of_strides_and_shapes():
    from rx_met_b200 import kept_codes
    dy, x = torch.randn(60, 80, device="cuda").to(torch.bfloat16), torch.randn(60, 100, device="cuda").to(torch.bfloat16)
    kept = kept_codes.keep(x)
    want = kept_codes.weight_gradient(dy, kept)
    odd = torch.empty(60 * 80 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(60, 80)
    odd.copy_(dy)
    pitched = torch.zeros(60, 83, device="cuda", dtype=torch.bfloat16)[:, :80]
    pitched.copy_(dy)
    for d in (odd, pitched, dy.t().contiguous().t()):
        assert torch.equal(kept_codes.weight_gradient(d, kept), want)
    deep = kept_codes.keep(x.view(3, 20, 100))
    assert torch.equal(kept_codes.weight_gradient(dy.view(3, 20, 80), deep), want)
    loose = kept_codes.KeptCodes(kept.codes.contiguous(), kept.exponents, kept.dtype)   # rows on 4 bytes
    assert torch.equal(kept_codes.weight_gradient(dy, loose), want)
    one = dy[:1].expand(60, 80)
    assert torch.equal(kept_codes.weight_gradient(one, kept), kept_codes.weight_gradient(one.contiguous(), kept))
    none = kept_codes.weight_gradient(dy[:0], kept_codes.keep(x[:0]))
    assert none.shape == (80, 100) and not none.any()


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_weight_gradient_of_what_is_not_finite(dtype):
    """A group that is not finite makes its columns NaN, a gradient that is not finite its row, and nothing else."""
    from rx_met_b200 import kept_codes
    dy, x = torch.randn(300, 80, device="cuda").to(dtype), torch.randn(300, 100, device="cuda").to(dtype)
    x[7, 40] = float("inf")
    dy[200, 11] = float("nan")
    got = kept_codes.weight_gradient(dy, kept_codes.keep(x))
    bad = torch.zeros(80, 100, device="cuda", dtype=torch.bool)
    bad[:, 32:64] = True
    bad[11] = True
    assert bool(torch.isnan(got[bad]).all()) and bool(torch.isfinite(got[~bad]).all())


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_weight_gradient_at_the_ends_of_the_number_range(dtype):
    """Products of the largest codes of the type's ends, each of them exact: one token an element."""
    from rx_met_b200 import kept_codes
    info = torch.finfo(dtype)
    tops = torch.tensor([info.max / 2, info.smallest_normal * 4, 1.0, 127 * 2.0 ** -24], device="cuda", dtype=torch.float64)
    for top in tops.tolist():
        x = torch.zeros(4, 32, device="cuda", dtype=dtype)
        for t in range(4):
            x[t, t] = top * (1 + t / 8)
        kept = kept_codes.keep(x)
        value = gl.values(*gl.keep(x))
        dy = (torch.randn(4, 16, device="cuda") / 4).to(dtype)
        got = kept_codes.weight_gradient(dy, kept, dtype=torch.float32)
        want = dy.double().T @ value
        # below the normal numbers the tensor cores may take an operand or a sum for zero: 2^-126 of it
        ml.within(got, want, want.abs() * 2.0 ** -22 + 2.0 ** -125)


@pytest.mark.parametrize("dtype", ml.TYPES)
def test_linear(dtype):
    from rx_met_b200 import kept_codes
    x, weight, bias = (t.to(dtype).requires_grad_() for t in (torch.randn(3, 50, 70, device="cuda"), torch.randn(90, 70, device="cuda") / 8, torch.randn(90, device="cuda")))
    dy = torch.randn(3, 50, 90, device="cuda").to(dtype)
    y = kept_codes.linear(x, weight, bias)
    assert torch.equal(y, torch.nn.functional.linear(x, weight, bias))
    dx, dweight, dbias = torch.autograd.grad(y, [x, weight, bias], dy)
    want_dx, want_dbias = torch.autograd.grad(torch.nn.functional.linear(x, weight, bias), [x, bias], dy)
    # the same products of torch's, which may choose another of its kernels
    assert torch.allclose(dx, want_dx, rtol=2 * ml.UNIT[dtype], atol=70 * 2.0 ** -20) and torch.allclose(dbias.double(), dy.double().sum(dim=(0, 1)), rtol=2 * ml.UNIT[dtype], atol=1e-4)
    value = gl.values(*gl.keep(x.detach())).flatten(0, 1)
    d = dy.flatten(0, 1)
    want, bound = d.double().T @ value, weight_bound(d, value, 150)
    ml.within(dweight, want, bound + (want.abs() + bound) * ml.UNIT[dtype] + ml.TINY[dtype])
    alone = torch.autograd.grad(kept_codes.linear(x.detach(), weight), weight, dy)[0]
    assert torch.equal(alone, dweight)
    assert torch.allclose(torch.autograd.grad(kept_codes.linear(x, weight.detach()), x, dy)[0], dx, rtol=2 * ml.UNIT[dtype], atol=70 * 2.0 ** -20)
    with torch.no_grad():
        assert torch.allclose(kept_codes.linear(x, weight), torch.nn.functional.linear(x, weight))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert kept_codes.linear(x, weight, bias).dtype == dtype


def test_what_is_kept_between_the_passes():
    """Codes in place of the activations: the memory that a graph holds."""
    from rx_met_b200 import kept_codes
    x = torch.randn(4096, 1024, device="cuda", dtype=torch.bfloat16).requires_grad_()
    weight = torch.randn(64, 1024, device="cuda", dtype=torch.bfloat16).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = kept_codes.gated_product(x, x)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held <= 2 * (4096 * 1024 + 4096 * 32) + 4096
    before = torch.cuda.memory_allocated()
    z = kept_codes.linear(x * 1, weight)
    assert torch.cuda.memory_allocated() - before <= 4096 * 1024 + 4096 * 32 + z.numel() * 2 + 4096


def test_graphs_streams_and_traces():
    from rx_met_b200 import kept_codes
    x, up = (torch.randn(300, 200, device="cuda").half().requires_grad_() for _ in range(2))
    weight = torch.randn(130, 200, device="cuda").half().requires_grad_()
    dy = torch.randn(300, 130, device="cuda").half()

    def step():
        y = kept_codes.linear(kept_codes.gated_product(x, up), weight)
        return [y.detach(), *torch.autograd.grad(y, [x, up, weight], dy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
    for call in (lambda t: kept_codes.values(kept_codes.keep(t)), lambda t: kept_codes.gated_product(t, t)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x.detach())


def test_refusals():
    from rx_met_b200 import kept_codes
    x = torch.zeros(4, 64, device="cuda")
    kept = kept_codes.keep(x)
    for call in (lambda: kept_codes.keep(x.double()), lambda: kept_codes.keep(x[:, :0]), lambda: kept_codes.keep(torch.zeros(2, 131072, device="cuda")),
                 lambda: kept_codes.values(kept._replace(codes=x)), lambda: kept_codes.values(kept._replace(exponents=kept.exponents[:, :1])),
                 lambda: kept_codes.values(kept._replace(exponents=kept.exponents.cpu())), lambda: kept_codes.gated_product(x, x[:, :63]),
                 lambda: kept_codes.gated_product(x, x.half()), lambda: kept_codes.gated_product(x, x.cpu()), lambda: kept_codes.weight_gradient(x[:3], kept),
                 lambda: kept_codes.weight_gradient(x.half(), kept), lambda: kept_codes.weight_gradient(x.cpu(), kept), lambda: kept_codes.weight_gradient(x, kept, dtype=torch.int8),
                 lambda: kept_codes.linear(x, x.half()), lambda: kept_codes.linear(x[0], x), lambda: kept_codes.linear(x, x[:, :63])):
        with pytest.raises(RuntimeError):
            call()
