"""Group normalization whose mean is far from zero: the error follows the spread,
not the mean.

All that the statistics add up are differences of values of the group to each
other, exact or rounded to 2^-24 of themselves, so the mean is off by at most 64
half steps of the mean difference (the constant of test_group_norm_gpu.py).  It is
kept as two fp32 numbers, 2^-48 of itself; 2^-36 leaves room for sums of a few
bits more than that.  Behind it come a difference, a product and a sum, half a step
of what they work on each: 2^-24 * 72 * (|x - mean| + mean |x - mean|) * rstd *
|gamma| + 2^-24 * 72 * |beta| in all."""
import pytest

from tests.token_ops import group_norm_64, group_norm_desc, joined, run_group_norm, split

pytestmark = pytest.mark.gpu

# held on chip by one block and by a cluster, read twice, and pixels that no vector load may use
SHAPES = [(1, 16, 16, 64, 64, 8), (2, 96, 96, 64, 64, 2), (1, 400, 300, 128, 128, 4),
          (2, 40, 30, 30, 30, 3), (1, 300, 200, 13, 17, 1)]


@pytest.mark.parametrize("value", [1000.1, -77.7, 123456.7])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_constant_groups(shape, value):
    """y is beta but for the mean's residue: 2^-36 |mean| / sqrt(eps) of gamma."""
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, c_store, groups = shape
    x = torch.full((n, h, w, c_store), value, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    gamma, beta = torch.randn(2, c, generator=g, device="cuda")
    y = torch.empty_like(x)
    run_group_norm(L, group_norm_desc(L, x.shape, c, groups, 1e-5, 0, 0, 0), x, gamma, beta, y)
    tol = 2.0 ** -36 * abs(value) * 1e-5 ** -0.5 * gamma.abs().double() + 2.0 ** -23 * beta.abs()
    err = (y[..., :c].double() - beta.double()).abs()
    assert (err <= tol + 2.0 ** -40).all(), float((err / tol).max())


@pytest.mark.parametrize("offset", [0.0, 1000.0, -1e5])
@pytest.mark.parametrize("kind", ["float32", "split"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_spread_about_a_far_mean(shape, kind, offset):
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, c_store, groups = shape
    if kind == "split" and c_store % 16:
        pytest.skip("split tensors hold a multiple of 16 channels per plane")
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.zeros(n, h, w, c_store, device="cuda")
    x[..., :c] = torch.randn(n, h, w, c, generator=g, device="cuda") + offset
    gamma, beta = torch.randn(2, c, generator=g, device="cuda")
    values = x[..., :c].double()
    xt = 0
    if kind == "split":
        x, xt = split(x, c_store), 3
        values = joined(x, c, c_store).float().double()  # hi + lo is taken in fp32
    y = torch.empty(n, h, w, c_store, device="cuda")
    d = group_norm_desc(L, y.shape, c, groups, 1e-5, 0, xt, 0)
    run_group_norm(L, d, x, gamma, beta, y)
    want, _ = group_norm_64(values, groups, gamma, beta, 1e-5, 0)
    v = values.reshape(n, h * w, groups, -1)
    mean = v.mean(dim=(1, 3), keepdim=True)
    far = (v - mean).abs()
    rstd = 1 / torch.sqrt((far ** 2).mean(dim=(1, 3), keepdim=True) + 1e-5)
    spread = ((far + far.mean(dim=(1, 3), keepdim=True)) * rstd).reshape(values.shape)
    residue = (2.0 ** -36 * mean.abs() * rstd).expand_as(v).reshape(values.shape)
    tol = 72 * 2.0 ** -24 * (spread * gamma.abs() + beta.abs()) + residue * gamma.abs() \
        + 2.0 ** -24 * want.abs()
    err = (y[..., :c].double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("outlier", [300.0, -1e4, 1e6])
@pytest.mark.parametrize("shape", SHAPES + [(1, 9, 40, 4096, 4096, 1)], ids=str)
def test_an_outlier_at_the_first_pixel(shape, outlier):
    """The value that a group's differences are taken to lies far from all others:
    64 half steps of the mean difference to it besides."""
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, c_store, groups = shape
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.zeros(n, h, w, c_store, device="cuda")
    x[..., :c] = torch.randn(n, h, w, c, generator=g, device="cuda") + 20.0
    x[:, 0, 0, :c:c // groups] = outlier
    gamma, beta = torch.randn(2, c, generator=g, device="cuda")
    y = torch.empty_like(x)
    run_group_norm(L, group_norm_desc(L, x.shape, c, groups, 1e-5, 0, 0, 0), x, gamma, beta, y)
    values = x[..., :c].double()
    want, _ = group_norm_64(values, groups, gamma, beta, 1e-5, 0)
    v = values.reshape(n, h * w, groups, -1)
    mean = v.mean(dim=(1, 3), keepdim=True)
    far = (v - mean).abs()
    rstd = 1 / torch.sqrt((far ** 2).mean(dim=(1, 3), keepdim=True) + 1e-5)
    base = (v - v[:, :1, :, :1]).abs().mean(dim=(1, 3), keepdim=True)
    spread = ((far + far.mean(dim=(1, 3), keepdim=True) + base) * rstd).reshape(values.shape)
    tol = 72 * 2.0 ** -24 * (spread * gamma.abs() + beta.abs()) + 2.0 ** -24 * want.abs()
    err = (y[..., :c].double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
