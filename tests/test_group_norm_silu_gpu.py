"""SiLU behind the group normalization: what one channel holds stays in that
channel (neighbours share a reciprocal in the kernels), and values far below
zero tend to zero.

Shapes: images held on chip, images read twice, and pixel strides that no vector
load may use."""
import pytest

from tests.token_ops import HALF_STEP, group_norm_64, group_norm_desc, joined, run_group_norm, split

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16", "split"]
IMAGES = [(2, 9, 7), (1, 400, 300)]


def check(y, want, size, half):
    """The tolerance of test_group_norm_gpu.py; a NaN is not within it."""
    err = (y.double() - want).abs()
    tol = half * want.abs() + 72 * 2.0 ** -24 * size + 2.0 ** -25
    assert (err <= tol).all(), float((err / tol).max())


def stored(xf, c_store, kind, garbage):
    """fp32 [..., c] -> (x of the type with `garbage` behind its channels, what x holds in 64
    bits)."""
    import torch
    c = xf.shape[-1]
    if kind == "split":
        x = split(xf, c_store)
        values = joined(x, c, c_store)
        x[..., c:c_store] = garbage
        x[..., c_store + c:] = garbage
        return x, values
    x = torch.full((*xf.shape[:-1], c_store), garbage, dtype=getattr(torch, kind), device="cuda")
    x[..., :c] = xf
    return x, x[..., :c].double()


def normal(shape, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    return x, 1 + 0.2 * torch.randn(shape[-1], generator=g, device="cuda"), \
        0.2 * torch.randn(shape[-1], generator=g, device="cuda")


@pytest.mark.parametrize("garbage", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("image", IMAGES, ids=str)
@pytest.mark.parametrize("c, c_store, groups", [(13, 16, 1), (15, 16, 15), (33, 48, 11)])
def test_padding_beside_an_odd_last_channel(c, c_store, groups, image, kind, garbage):
    import torch
    from computeengine_b200 import _lib as L
    xf, gamma, beta = normal((*image, c), 1)
    x, values = stored(xf, c_store, kind, float(garbage))
    y = torch.full((*image, c_store), 7.0, device="cuda")
    d = group_norm_desc(L, (*image, c_store), c, groups, 1e-5, L.IE_ACT_SILU, TYPES.index(kind),
                        L.IE_DT_F32)
    run_group_norm(L, d, x, gamma, beta, y)
    want, size = group_norm_64(values, groups, gamma, beta, 1e-5, 3)
    check(y[..., :c], want, size, HALF_STEP[torch.float32])
    assert not y[..., c:].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("image", IMAGES, ids=str)
@pytest.mark.parametrize("per_group", [1, 3, 5])
def test_a_group_that_is_nan_stays_alone(per_group, image, kind):
    """Groups with an odd number of channels: one holds a NaN, another an infinity."""
    import torch
    from computeengine_b200 import _lib as L
    c = 16 * per_group
    xf, gamma, beta = normal((*image, c), 2)
    lost = [2, 9]
    for g, v in zip(lost, (float("nan"), float("inf"))):
        xf[0, 3, 4, g * per_group] = v
    x, values = stored(xf, c, kind, 0.0)
    if kind == "split":  # inf - inf in the lo plane
        values = values.float().double()
    y = torch.full((*image, c), 7.0, device="cuda")
    d = group_norm_desc(L, (*image, c), c, 16, 1e-5, L.IE_ACT_SILU, TYPES.index(kind), L.IE_DT_F32)
    run_group_norm(L, d, x, gamma, beta, y)
    want, size = group_norm_64(values, 16, gamma, beta, 1e-5, 3)
    bad = torch.zeros(image[0], 16, dtype=torch.bool, device="cuda")
    bad[0, lost] = True
    bad = bad.repeat_interleave(per_group, 1)[:, None, None].expand(y.shape)
    assert torch.isnan(y[bad]).all()
    check(y[~bad], want[~bad], size[~bad], HALF_STEP[torch.float32])


@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("image", IMAGES, ids=str)
def test_nan_in_gamma_and_beta_stays_in_its_channel(image, act):
    import torch
    from computeengine_b200 import _lib as L
    x, gamma, beta = normal((*image, 32), 3)
    gamma[4] = beta[11] = float("nan")
    y = torch.empty_like(x)
    run_group_norm(L, group_norm_desc(L, x.shape, 32, 4, 1e-5, act, 0, 0), x, gamma, beta, y)
    want, size = group_norm_64(x.double(), 4, gamma, beta, 1e-5, act)
    assert torch.isnan(y[..., [4, 11]]).all()
    rest = [i for i in range(32) if i not in (4, 11)]
    check(y[..., rest], want[..., rest], size[..., rest], HALF_STEP[torch.float32])


@pytest.mark.parametrize("c_store", [64, 65])
@pytest.mark.parametrize("image", IMAGES, ids=str)
def test_far_below_zero(image, c_store):
    """gamma is 0, so z is beta.  The exponent -z log2 e is off by 2^-24 of itself
    for the product and 2^-25 for the constant, the exponential, the sum, the
    reciprocals and the products by a few half steps (16 cover them): relative
    2^-24 (16 + 1.5 |z|).  From z = -87 on the denominator's reciprocal is no
    normal number any more; |z| e^z is below 2^-118 there and may be 0."""
    import torch
    from computeengine_b200 import _lib as L
    x = torch.zeros(*image, c_store, device="cuda")
    x[..., :64] = normal((*image, 64), 4)[0]
    z = -torch.linspace(1, 87, 64, device="cuda")
    z[::7] = torch.tensor([-1e25, -1e20, -100.0, -88.5, -1000.0, -3e38, -5e4, -43.0, -1e30, -200.0],
                          device="cuda")
    beta = z.clone()
    y = torch.empty_like(x)
    d = group_norm_desc(L, x.shape, 64, 8, 1e-5, L.IE_ACT_SILU, 0, 0)
    run_group_norm(L, d, x, torch.zeros(64, device="cuda"), beta, y)
    z = z.double()
    want = z * torch.sigmoid(z)
    tol = want.abs() * 2.0 ** -24 * (16 + 1.5 * z.abs())
    tol[z < -87] = 2.0 ** -118
    err = (y[..., :64].double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())
