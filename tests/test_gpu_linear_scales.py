"""MatMulNBits with scales at the ends of their range: 16-bit rows, few and many, against the definition in 64 bits."""
import math

import numpy as np
import pytest

import decoder_oracle as D
import test_gpu_decoder as G

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def check_scales(rows, k, n, group, kind, scales, x_size, zero_points, bias, seed, silent=None):
    """Scales f32 [n][groups]; x of about `x_size`, 0 in the groups of `silent`.  Bound: the result's rounding, a rounding of
    each weight to the type's precision, and the f32 sums: that the scales are far from 1 changes none of these.  A weight that is
    tiny beside the largest of its output may lose 2^-36 of that one."""
    g = torch.Generator().manual_seed(seed)
    w = D.linear_weights(g, n, k, group, zero_points, bias)
    w["scales"] = scales.astype(np.float32)
    if bias:
        w["bias"] *= float(np.abs(w["scales"]).max()) * x_size
    x = torch.randn(rows, k, generator=g) * x_size
    for b in silent or ():
        x[:, b * group : (b + 1) * group] = 0
    x = x.to(D.TYPES[kind])
    y = torch.full((rows, n), math.nan, dtype=x.dtype, device="cuda")
    s = G.session([G.linear_node(k, n, group, w)], {"x": x.cuda()}, {"y": y}, w)
    G.run(s)
    want, h = D.linear(x, w, k), D.half_step(kind)
    size = x.double().abs() @ D.linear_matrix(w, k).abs().t()
    floor = x.double().abs().sum(-1, keepdim=True) * torch.from_numpy(np.abs(w["scales"]).max(-1)).double()[None] * 2.0**-36
    if silent:  # beside a scale that far away nothing may be lost
        floor = 0.0
    extra = torch.from_numpy(w["bias"]).double().abs() * 2.0**-23 if bias else 0.0
    assert torch.isfinite(want.to(x.dtype)).all() and (want.abs() > torch.finfo(x.dtype).tiny).double().mean() > 0.9, "the case is about weights, not about results out of range"
    G.within(y, want, D.rounding(kind, want) + ((k + 2) * 2.0**-23 + h) * (1 + h) * size + floor + extra)
    first = y.clone()
    G.run(s)
    assert torch.equal(first, y)
    return s


def spread(n, blocks, low, high, seed, kind=np.float32):
    """Scales over a range, their logarithms even; every output has its own part of it."""
    g = np.random.default_rng(seed)
    middle = g.uniform(math.log(low), math.log(high), (n, 1))
    return np.exp(np.clip(middle + g.uniform(-1, 1, (n, blocks)), math.log(low), math.log(high))).astype(kind).astype(np.float32)


@pytest.mark.parametrize("rows", [5, 16, 17, 40, 300])
@pytest.mark.parametrize("group", [16, 32, 128])
@pytest.mark.parametrize("low,high,x_size,kind", [(4000, 30000, 1e-3, "float16"), (2e-9, 3e-8, 1e3, "float16"), (1e-7, 4e-5, 30.0, "float16"), (1e-3, 1e-1, 1.0, "float16"),
                                                  (4e37, 3e38, 1e-4, "bfloat16"), (1e-30, 1e-25, 1.0, "bfloat16"), (1e-3, 1e-1, 1.0, "bfloat16")])
def test_linear_scales_of_any_size(rows, group, low, high, x_size, kind):
    """f32 scales whose products with a code leave the 16-bit type's range, or its normal numbers."""
    k, n = 270, 150
    check_scales(rows, k, n, group, kind, spread(n, -(-k // group), low, high, rows + group), x_size, rows % 2 == 1, rows == 40, rows)


@pytest.mark.parametrize("rows,n", [(17, 96), (129, 520), (1000, 70)])
def test_linear_scales_of_f16_that_overflow_with_a_code(rows, n):
    check_scales(rows, 128, n, 32, "float16", spread(n, 4, 3000, 60000, rows, np.float16), 1e-3, True, rows == 129, rows)


def test_linear_with_every_output_its_own_size():
    """Outputs next to one another whose scales lie 2^40 apart, negative and zero scales among them."""
    scales = spread(200, 4, 1e-9, 1e2, 1)
    scales[::7] *= -1
    scales[3], scales[5, 1] = 0, 0
    for rows in (16, 64, 257):
        g = torch.Generator().manual_seed(rows)
        w = D.linear_weights(g, 200, 128, 32, True, False)
        w["scales"] = scales
        x = torch.randn(rows, 128, generator=g).half()
        y = torch.full((rows, 200), math.nan, dtype=torch.float16, device="cuda")
        G.run(G.session([G.linear_node(128, 200, 32, w)], {"x": x.cuda()}, {"y": y}, w))
        want, h = D.linear(x, w, 128), D.half_step("float16")
        size = x.double().abs() @ D.linear_matrix(w, 128).abs().t()
        G.within(y, want, D.rounding("float16", want) + (130 * 2.0**-23 + h) * (1 + h) * size + 1e-30)


@pytest.mark.parametrize("rows", [16, 20, 40, 200])
@pytest.mark.parametrize("kind,low,high", [("float16", 1e-8, 1e3), ("bfloat16", 1e-38, 1e8)])
def test_linear_groups_of_one_output_far_apart(rows, kind, low, high):
    """A group whose scale is far below another's of the same output, of which x shows nothing."""
    scales = np.full((70, 5), low, np.float32)
    scales[:, 2] = high
    scales[1::2, :] *= np.float32(1.00001)
    check_scales(rows, 300, 70, 64, kind, scales, 1e3 if kind == "float16" else 1e5, rows == 20, False, rows, silent=[2])


@pytest.mark.parametrize("rows", [4, 33])
def test_linear_scales_that_are_no_numbers(rows):
    """An infinite or NaN scale concerns its own output alone."""
    w = D.linear_weights(torch.Generator().manual_seed(rows), 80, 64, 32, False, False)
    w["weights"][:] = 0x99
    w["scales"][3, 0], w["scales"][50, 1] = math.inf, math.nan
    x = torch.rand(rows, 64, generator=torch.Generator().manual_seed(rows)).half() + 1
    y = torch.zeros(rows, 80, dtype=torch.float16, device="cuda")
    G.run(G.session([G.linear_node(64, 80, 32, w)], {"x": x.cuda()}, {"y": y}, w))
    rest = [i for i in range(80) if i not in (3, 50)]
    assert torch.isinf(y[:, 3]).all() and torch.isnan(y[:, 50]).all() and torch.isfinite(y[:, rest]).all()
