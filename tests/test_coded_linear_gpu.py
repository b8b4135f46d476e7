"""Product of 8-bit codes on the GPU against its formula in 64 bits: sums are exact, the epilogue is bounded by its roundings."""
import pytest
import torch

import mixer_lib as ml

pytestmark = pytest.mark.gpu


def padded(codes):
    held = torch.zeros(codes.shape[0], (codes.shape[1] + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    held[:, :codes.shape[1]] = codes
    return held[:, :codes.shape[1]]


def problem(rows, inner, outer, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(-127, 128, (rows, inner), device="cuda", generator=g).to(torch.int8)
    weight = torch.randint(-127, 128, (outer, inner), device="cuda", generator=g).to(torch.int8)
    scale = torch.rand(rows, device="cuda", generator=g) * 0.02 + 0.01
    weight_scale = (torch.rand(outer, device="cuda", generator=g) + 0.5) / (127 * inner ** 0.5)
    bias = torch.randn(outer, device="cuda", generator=g)
    residual = torch.randn(rows, outer, device="cuda", generator=g).to(dtype)
    return codes, scale, weight, weight_scale, bias, residual


def check(codes, scale, weight, weight_scale, bias, activation, residual, dtype):
    from rx_met_b200.coded_linear import CodedWeight, coded_linear
    got = coded_linear(codes, scale, CodedWeight(weight, weight_scale), bias=bias, activation=activation, residual=residual, dtype=dtype)
    want, magnitude = ml.linear(codes, scale, weight, weight_scale, bias, activation, residual)
    assert got.dtype == dtype
    # six roundings in 32 bits up to the activation (its slope is below 1.13), eight units for the activation's functions
    ml.within(got, want, want.abs() * ml.UNIT[dtype] * 1.01 + magnitude * 16 * 2.0 ** -24 + ml.TINY[dtype])
    return got


SHAPES = [(1, 1, 1), (1, 16, 8), (1, 1024, 4096), (2, 100, 77), (3, 333, 1000), (8, 512, 256), (9, 256, 130), (17, 1040, 96), (33, 64, 640), (64, 128, 128),
          (100, 2048, 200), (128, 48, 129), (129, 80, 1100), (257, 1000, 384), (500, 4096, 512), (1000, 144, 3000)]


@pytest.mark.parametrize("rows,inner,outer", SHAPES)
@pytest.mark.parametrize("dtype", ml.TYPES)
def test_product(rows, inner, outer, dtype):
    codes, scale, weight, weight_scale, bias, residual = problem(rows, inner, outer, seed=rows + inner, dtype=dtype)
    full = check(padded(codes), scale, padded(weight), weight_scale, bias, "none", residual, dtype)
    if rows * outer < 200_000:   # the same for rows that do not start on 16 bytes
        assert torch.equal(full, check(codes, scale, weight, weight_scale, bias, "none", residual, dtype))


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("with_residual", [True, False])
def test_epilogue(rows, activation, with_bias, with_residual):
    codes, scale, weight, weight_scale, bias, residual = problem(rows, 96, 200, seed=rows)
    check(padded(codes), scale, padded(weight), weight_scale, bias if with_bias else None, activation, residual if with_residual else None, torch.float32)


@pytest.mark.parametrize("rows", [1, 4, 30, 200])
def test_extreme_codes(rows):
    """The largest sums that 8-bit codes can make, at the largest inner size, and scales that overflow or are not finite."""
    inner = 131071
    codes = torch.full((rows, inner), -128, dtype=torch.int8, device="cuda")
    weight = torch.full((3, inner), -128, dtype=torch.int8, device="cuda")
    weight[1] = 127
    one = torch.ones(rows, device="cuda")
    got = check(padded(codes), one, padded(weight), torch.ones(3, device="cuda"), None, "none", None, torch.float32)
    assert float(got[0, 0]) == float(torch.tensor(128.0 * 128.0 * inner))
    from rx_met_b200.coded_linear import CodedWeight, coded_linear
    bad = one.clone()
    bad[0] = float("nan")
    out = coded_linear(padded(codes), bad, CodedWeight(padded(weight), torch.ones(3, device="cuda")), activation="relu", dtype=torch.float32)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()


@pytest.mark.parametrize("aligned", [True, False])
def test_many_rows(aligned):
    """More rows than a grid's axis has places for the smallest tiles; a few of them are compared."""
    from rx_met_b200.coded_linear import CodedWeight, coded_linear
    rows = 1_100_000 if aligned else 300_000
    inner = 32 if aligned else 33
    codes = torch.randint(-127, 128, (rows, inner), device="cuda", dtype=torch.int8)
    weight = torch.randint(-127, 128, (5, inner), device="cuda", dtype=torch.int8)
    out = coded_linear(codes, torch.ones(rows, device="cuda"), CodedWeight(weight, torch.ones(5, device="cuda")), dtype=torch.float32)
    at = torch.cat([torch.arange(300, device="cuda"), torch.arange(rows - 300, rows, device="cuda"), torch.randint(0, rows, (2000,), device="cuda")])
    assert torch.equal(out[at].double(), codes[at].double() @ weight.double().T)


def test_strides_and_leading_dimensions():
    from rx_met_b200.coded_linear import CodedWeight, code_weight, coded_linear
    codes, scale, weight, weight_scale, bias, residual = problem(60, 100, 50, dtype=torch.bfloat16)
    w = CodedWeight(padded(weight), weight_scale)
    base = coded_linear(padded(codes), scale, w, bias=bias, residual=residual)
    shaped = coded_linear(padded(codes).view(3, 20, 100), scale.view(3, 20), w, bias=bias, residual=residual.view(3, 20, 50))
    assert shaped.shape == (3, 20, 50) and torch.equal(shaped.view(60, 50), base)
    wide = torch.zeros(60, 77, dtype=torch.bfloat16, device="cuda")
    wide[:, 13:63] = residual
    assert torch.equal(coded_linear(padded(codes), scale, w, bias=bias, residual=wide[:, 13:63]), base)
    assert torch.equal(coded_linear(padded(codes)[::2], scale[::2], w, bias=bias, residual=residual[::2]), base[::2])
    column = codes.t().contiguous().t()
    assert torch.equal(coded_linear(column, scale, w, bias=bias, residual=residual), base)
    assert coded_linear(padded(codes)[:0], scale[:0], w).shape == (0, 50)
    assert torch.equal(coded_linear(padded(codes)[7], scale[7], w, bias=bias, residual=residual[7]), base[7])
    x = torch.randn(50, 100, device="cuda")
    coded = code_weight(x)
    assert bool(((coded.codes.double() * coded.scale.double()[:, None] - x.double()).abs() <= coded.scale.double()[:, None] * 0.51).all())


def test_refusals():
    from rx_met_b200.coded_linear import CodedWeight, coded_linear
    codes, scale, weight, weight_scale, bias, residual = problem(4, 32, 16)
    w = CodedWeight(weight, weight_scale)
    bad = [dict(codes=codes.int()), dict(codes=codes[:, :31]), dict(scale=scale[:3]), dict(scale=scale.double()), dict(weight=CodedWeight(weight, weight_scale[:3])),
           dict(weight=CodedWeight(weight.float(), weight_scale)), dict(bias=bias[:2]), dict(residual=residual.half()), dict(residual=residual[:2]),
           dict(dtype=torch.float64), dict(codes=codes.cpu()), dict(weight=CodedWeight(weight.cpu(), weight_scale)),
           dict(codes=torch.zeros(4, 131072, dtype=torch.int8, device="cuda"), weight=CodedWeight(torch.zeros(16, 131072, dtype=torch.int8, device="cuda"), weight_scale), residual=None)]
    for change in bad:
        arguments = dict(dict(codes=codes, scale=scale, weight=w, bias=bias, residual=residual, dtype=torch.float32), **change)
        with pytest.raises(RuntimeError):
            coded_linear(arguments.pop("codes"), arguments.pop("scale"), arguments.pop("weight"), **arguments)
    with pytest.raises(ValueError):
        coded_linear(codes, scale, w, activation="swish")
