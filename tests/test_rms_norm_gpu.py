"""Residual norm on the GPU against its formula in 64 bits: output, codes, gradients, odd sizes and strides, refusals."""
import pytest
import torch

import mixer_lib as ml

pytestmark = pytest.mark.gpu

# 32-bit sums: a lane adds at most 16 elements in order, lanes and warps add in a tree of ten steps; square, mean, root, two products
ROUNDINGS = (16 + 10 + 8) * 2.0 ** -24


def tensors(rows, width, dtype, seed=0, pitch=None, weight_type=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda: torch.randn(rows, pitch or width, device="cuda", generator=g).to(dtype)[:, :width]  # noqa: E731
    weight = (1 + 0.1 * torch.randn(width, device="cuda", generator=g)).to(weight_type)
    return make(), weight, make()


SHAPES = [(1, 1), (1, 8), (3, 7), (1, 1024), (5, 100), (2, 4096), (300, 257), (777, 512), (9, 1001), (1000, 64), (4, 16384), (3, 16383), (2000, 2048)]


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_norm(rows, width, dtype, with_residual):
    from rx_met_b200 import rms_norm
    x, weight, residual = tensors(rows, width, dtype)
    residual = residual if with_residual else None
    y, total = rms_norm.add_rms_norm(x, weight, residual, 1e-5)
    want, wanted_total, _ = ml.norm(x, weight, residual, 1e-5)
    assert y.dtype == dtype and total.dtype == dtype
    ml.within(y, want, want.abs() * (ml.UNIT[dtype] + ROUNDINGS) * 1.01 + ml.TINY[dtype])
    ml.within(total, wanted_total, wanted_total.abs() * (ml.UNIT[dtype] + 2.0 ** -23) * 1.01 + ml.TINY[dtype])


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("rows,width", SHAPES)
def test_codes(rows, width, dtype):
    from rx_met_b200 import rms_norm
    x, weight, residual = tensors(rows, width, dtype, seed=1)
    codes, scale, total = rms_norm.add_rms_norm_codes(x, weight, residual, 1e-5)
    want, wanted_total, _ = ml.norm(x, weight, residual, 1e-5)
    top = want.abs().amax(dim=1) / 127
    ml.within(scale, top, top * (ROUNDINGS + 2.0 ** -23))
    # half a step, and what y and the quotient by the scale are off by at 127 steps
    ml.within(codes.double() * scale.double()[:, None], want, (top * (0.5 + 127 * (3 * ROUNDINGS + 2.0 ** -21)))[:, None].expand_as(want))
    assert codes.dtype == torch.int8 and int(codes.abs().max()) == 127
    assert codes.stride(0) % 16 == 0 or rows == 1
    ml.within(total, wanted_total, wanted_total.abs() * (ml.UNIT[dtype] + 2.0 ** -23) * 1.01 + ml.TINY[dtype])


def test_codes_of_rows_and_odd_rows():
    from rx_met_b200 import rms_norm
    x = torch.randn(6, 50, device="cuda")
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 0
    x[4, 49] = -3.0
    codes, scale = rms_norm.code_rows(x)
    assert torch.equal(scale[[0, 5]], (x[[0, 5]].double().abs().amax(dim=1) / 127).float())   # one rounding of the quotient
    assert scale[1] == 0 and not codes[1].any()
    assert torch.isnan(scale[2]) and torch.isinf(scale[3])
    assert codes[4, 49] == -127 and not codes[4, :49].any()
    for row in (0, 5):
        step = scale[row].double()
        assert bool(((codes[row].double() * step - x[row].double()).abs() <= step * (0.5 + 127 * 2.0 ** -22)).all())


@pytest.mark.parametrize("dtype", ml.TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (300, 257), (777, 512), (5000, 64), (4, 16384), (2000, 2048), (33, 16383)])
@pytest.mark.parametrize("weight_type", [torch.float32, None])
@pytest.mark.parametrize("with_total", [True, False])
def test_gradients(rows, width, dtype, weight_type, with_total):
    from rx_met_b200 import rms_norm
    weight_type = weight_type or dtype
    x, weight, residual = (t.requires_grad_() for t in tensors(rows, width, dtype, seed=2, weight_type=weight_type))
    dy = torch.randn(rows, width, device="cuda").to(dtype)
    dtotal = torch.randn(rows, width, device="cuda").to(dtype) if with_total else None
    y, total = rms_norm.add_rms_norm(x, weight, residual, 1e-5)
    dx, dresidual, dweight = torch.autograd.grad([y, total] if with_total else [y], [x, residual, weight], [dy, dtotal] if with_total else [dy])
    assert dx.dtype == dtype and dweight.dtype == weight_type and torch.equal(dx, dresidual)
    _, _, rms = ml.norm(x.detach(), weight.detach(), residual.detach(), 1e-5)
    exact = x.detach().double() + residual.detach().double()
    want, wanted_weight = ml.norm_gradients(dy, dtotal, exact, weight.detach(), rms)
    d = (dy.double() * weight.detach().double()).abs()
    u = (exact * rms).abs()
    magnitude = rms * (d + u * (d * u).mean(dim=1, keepdim=True)) + (0 if dtotal is None else dtotal.double().abs())
    ml.within(dx, want, want.abs() * ml.UNIT[dtype] * 1.01 + magnitude * 3 * ROUNDINGS + ml.TINY[dtype])
    summed = (dy.double().abs() * u).sum(dim=0)
    # a CTA's rows in order, the CTAs in 32 strands
    ml.within(dweight, wanted_weight, wanted_weight.abs() * ml.UNIT[weight_type] * 1.01 + summed * (rows / 32 + 64) * 2.0 ** -24 + ml.TINY[weight_type])


# rows of which three arrays fit shared memory, or none; all by groups and by elements, with more rows than CTAs take at once
@pytest.mark.parametrize("rows,width,dtype", [(650, 8192, torch.float32), (650, 7201, torch.float32), (40, 9000, torch.float32), (40, 12001, torch.float32), (650, 15000, torch.float16),
                                              (650, 8191, torch.bfloat16), (650, 16381, torch.bfloat16)])
@pytest.mark.parametrize("with_total", [True, False])
def test_gradients_of_wide_rows(rows, width, dtype, with_total):
    test_gradients(rows, width, dtype, None, with_total)


def test_gradients_without_a_residual_or_a_trained_weight():
    from rx_met_b200 import rms_norm
    x, weight, residual = tensors(70, 96, torch.float32, seed=4)
    dy = torch.randn(70, 96, device="cuda")
    _, total, rms = ml.norm(x, weight, None, 1e-5)
    want, wanted_weight = ml.norm_gradients(dy, None, total, weight, rms)
    leaf, trained = x.clone().requires_grad_(), weight.clone().requires_grad_()
    dx, dweight = torch.autograd.grad(rms_norm.add_rms_norm(leaf, trained, None, 1e-5)[0], [leaf, trained], dy)
    assert torch.allclose(dx.double(), want, rtol=1e-5, atol=1e-5) and torch.allclose(dweight.double(), wanted_weight, rtol=1e-5, atol=1e-4)
    alone = torch.autograd.grad(rms_norm.add_rms_norm(leaf, weight, None, 1e-5)[0], leaf, dy)[0]
    assert torch.equal(alone, dx)
    both = [x.clone().requires_grad_(), residual.clone().requires_grad_()]
    grads = torch.autograd.grad(rms_norm.add_rms_norm(both[0], weight, both[1], 1e-5)[0], both, dy)
    assert torch.equal(grads[0], grads[1])
    only = torch.autograd.grad(rms_norm.add_rms_norm(x, weight, both[1], 1e-5)[0], both[1], dy)[0]
    assert torch.equal(only, grads[1])


def test_gradient_against_differences():
    from rx_met_b200 import rms_norm
    x, weight, residual = (t.requires_grad_() for t in tensors(4, 33, torch.float32, seed=3))
    a, b = torch.randn(4, 33, device="cuda"), torch.randn(4, 33, device="cuda")

    def loss(*leaves):
        y, total = rms_norm.add_rms_norm(leaves[0], leaves[1], leaves[2], 1e-5)
        return (y.double() * a).sum() + (total.double() * b).sum()

    leaves = [x, weight, residual]
    for i, g in enumerate(torch.autograd.grad(loss(*leaves), leaves)):
        way = torch.randn_like(leaves[i])
        h = 1e-2
        ends = [loss(*[t.detach() + (s * h * way if j == i else 0) for j, t in enumerate(leaves)]) for s in (1, -1)]
        slope, want = float(ends[0] - ends[1]) / (2 * h), float((g.double() * way).sum())
        # third derivative times h^2 / 6, and 132 outputs off by 1e-6 over 2 h
        assert abs(slope - want) <= 2e-3 * max(1.0, float((g.double() * way).abs().sum())), (slope, want)


def test_strides_shapes_and_reproducibility():
    from rx_met_b200 import rms_norm
    x, weight, residual = tensors(40, 256, torch.bfloat16, pitch=300)
    y, total = rms_norm.add_rms_norm(x, weight, residual)
    y2, total2 = rms_norm.add_rms_norm(x.contiguous().view(5, 8, 256), weight, residual.contiguous().view(5, 8, 256))
    assert y2.shape == (5, 8, 256) and torch.equal(y, y2.view(40, 256)) and torch.equal(total, total2.view(40, 256))
    y3, _ = rms_norm.add_rms_norm(x.t().contiguous().t(), weight, residual)   # elements of a row apart
    assert torch.equal(y, y3)
    odd = torch.empty(40 * 256 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(40, 256)   # off the 16-byte grid
    odd.copy_(x)
    ml.within(rms_norm.add_rms_norm(odd, weight, residual)[0], y.double(), y.double().abs() * 2.0 ** -7)
    codes, scale, _ = rms_norm.add_rms_norm_codes(x.view(40, 256)[:, :100], weight[:100])
    assert codes.shape == (40, 100) and scale.shape == (40,)
    empty = rms_norm.add_rms_norm(x[:0], weight, residual[:0])
    assert empty[0].shape == (0, 256)
    x, weight, residual = (t.requires_grad_() for t in tensors(5000, 1000, torch.float16))
    grads = [torch.autograd.grad(rms_norm.add_rms_norm(x, weight, residual)[0], [x, weight], torch.ones_like(x)) for _ in range(3)]
    assert all(torch.equal(a, b) for g in grads[1:] for a, b in zip(g, grads[0]))
    none = rms_norm.add_rms_norm(x[:0], weight, residual[:0])[0]
    assert not torch.autograd.grad(none.sum(), weight)[0].any()
    only_total = torch.autograd.grad(rms_norm.add_rms_norm(x, weight, residual)[1], [x, residual], torch.ones_like(x))
    assert all(bool((g == 1).all()) for g in only_total)


def test_refusals():
    from rx_met_b200 import rms_norm
    x, weight, residual = tensors(4, 64, torch.bfloat16)
    for call in (lambda: rms_norm.add_rms_norm(x, weight[:63], residual), lambda: rms_norm.add_rms_norm(x, weight, residual[:3]),
                 lambda: rms_norm.add_rms_norm(x, weight, residual.half()), lambda: rms_norm.add_rms_norm(x.double(), weight),
                 lambda: rms_norm.add_rms_norm(x, weight.cpu(), residual), lambda: rms_norm.add_rms_norm(torch.zeros(2, 16385, device="cuda"), torch.ones(16385, device="cuda")),
                 lambda: rms_norm.code_rows(torch.zeros(2, 0, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
