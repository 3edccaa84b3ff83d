"""ie_cuda_group_norm_nhwc against the definition in 64 bits.

Tolerance: z = (x - mean) * rstd * gamma + beta in fp32.  Each of the five
operations is off by half a step of what it works on, at most
2^-24 * (|x| + mean |x|) * rstd * |gamma| + 2^-24 |beta|; the mean and the
variance are sums whose partial sums are joined in trees and short chains, off
by a few dozen half steps at most: 64 half steps cover both.  An activation's
slope is at most 1.13, its own fp32 arithmetic is off by a few half steps of
|z|.  Then one rounding to the output type."""
import pytest

from tests.token_ops import (HALF_STEP, group_norm_64, group_norm_desc, joined, run_group_norm,
                             split)

pytestmark = pytest.mark.gpu


def check(y, want, size, half):
    err = (y.double() - want).abs()
    tol = half * want.abs() + 72 * 2.0 ** -24 * size + 2.0 ** -25
    assert not (err > tol).any(), float((err / tol).max())


def inputs(shape, seed, offset=0.5):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = shape[-1]
    x = torch.randn(shape, generator=g, device="cuda")
    x = x * (torch.rand(c, generator=g, device="cuda") + 0.5)
    x = x + offset * torch.randn(c, generator=g, device="cuda")
    gamma = 1 + 0.2 * torch.randn(c, generator=g, device="cuda")
    beta = 0.2 * torch.randn(c, generator=g, device="cuda")
    return x, gamma, beta


# small, odd and prime extents, one pixel, one channel per group, all channels
# in one group, groups that end inside a vector of channels, many images, and
# images of the sizes where the kernel changes
SHAPES = [
    (1, 1, 1, 32, 32), (1, 1, 1, 32, 1), (3, 1, 1, 7, 7), (2, 5, 3, 30, 3), (1, 7, 7, 1, 1),
    (1, 8, 8, 256, 32), (2, 64, 64, 320, 32), (5, 9, 13, 48, 4), (1, 33, 31, 40, 8),
    (40, 4, 4, 96, 32), (1, 128, 128, 64, 1), (2, 56, 56, 256, 32), (1, 256, 200, 24, 4),
    (1, 17, 19, 1280, 32), (1, 16, 16, 2048, 1), (3, 127, 129, 16, 16), (1, 400, 300, 128, 32),
    (1, 64, 64, 1000, 8), (300, 3, 5, 64, 4),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("act", range(5))
def test_shapes_and_activations(shape, act):
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, groups = shape
    x, gamma, beta = inputs((n, h, w, c), 1)
    y = torch.full_like(x, float("nan"))
    d = group_norm_desc(L, x.shape, c, groups, 1e-5, act, L.IE_DT_F32, L.IE_DT_F32)
    run_group_norm(L, d, x, gamma, beta, y)
    want, size = group_norm_64(x.double(), groups, gamma, beta, 1e-5, act)
    check(y, want, size, HALF_STEP[torch.float32])


TYPES = ["float32", "bfloat16", "float16", "split"]


@pytest.mark.parametrize("yt", TYPES)
@pytest.mark.parametrize("xt", TYPES)
@pytest.mark.parametrize("shape", [(2, 24, 24, 80, 96, 8), (1, 150, 160, 120, 128, 4),
                                   (1, 400, 300, 64, 64, 16)], ids=str)
def test_types_and_padding_channels(shape, xt, yt):
    """Every pair of types; stored channels past c hold garbage in x, zeros in y."""
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, c_store, groups = shape
    xf, gamma, beta = inputs((n, h, w, c), 2)
    code = {t: i for i, t in enumerate(TYPES)}
    if xt == "split":
        x = split(xf, c_store)
        xd = joined(x, c, c_store)
        x[..., c:c_store] = float("nan")
        x[..., c_store + c:] = float("nan")
    else:
        x = torch.full((n, h, w, c_store), float("nan"), dtype=getattr(torch, xt), device="cuda")
        x[..., :c] = xf
        xd = x[..., :c].double()
    planes = 2 if yt == "split" else 1
    dt = torch.bfloat16 if yt == "split" else getattr(torch, yt)
    y = torch.full((n, h, w, planes * c_store), float("nan"), dtype=dt, device="cuda")
    d = group_norm_desc(L, (n, h, w, c_store), c, groups, 1e-5, 3, code[xt], code[yt])
    run_group_norm(L, d, x, gamma, beta, y)
    want, size = group_norm_64(xd, groups, gamma, beta, 1e-5, 3)
    if yt == "split":  # the lo plane rounds what the hi plane left
        check(joined(y, c, c_store), want, size, 2.0 ** -16)
        assert not y[..., c:c_store].any() and not y[..., c_store + c:].any()
    else:
        check(y[..., :c], want, size, HALF_STEP[dt])
        assert not y[..., c:].any()


@pytest.mark.parametrize("c, c_store, shift", [(30, 30, 0), (24, 24, 2), (13, 17, 1), (64, 64, 4)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_any_alignment(c, c_store, shift, dtype):
    """Pixel strides and pointers that no vector load may use."""
    import torch
    from computeengine_b200 import _lib as L
    dt = getattr(torch, dtype)
    n, h, w, groups = 2, 70, 33, 1
    xf, gamma, beta = inputs((n, h, w, c), 3)
    count = n * h * w * c_store
    x = torch.zeros(count + shift, dtype=dt, device="cuda")[shift:].view(n, h, w, c_store)
    x[..., :c] = xf
    flat = torch.full((count + shift + 64,), 7.0, dtype=dt, device="cuda")
    y = flat[shift:shift + count].view(n, h, w, c_store)
    d = group_norm_desc(L, x.shape, c, groups, 1e-5, 4, *[{"float32": 0, "bfloat16": 1}[dtype]] * 2)
    run_group_norm(L, d, x, gamma, beta, y)
    want, size = group_norm_64(x[..., :c].double(), groups, gamma, beta, 1e-5, 4)
    check(y[..., :c], want, size, HALF_STEP[dt])
    assert (flat[:shift] == 7).all() and (flat[shift + count:] == 7).all()


@pytest.mark.parametrize("shape", [(1, 8, 8, 64, 8), (2, 64, 64, 320, 32), (1, 400, 300, 128, 4)],
                         ids=str)
def test_no_scale_in_place_and_repeat(shape):
    """NULL gamma and beta, y == x, and the same bytes every time."""
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, groups = shape
    x = inputs((n, h, w, c), 4)[0].bfloat16()
    want, size = group_norm_64(x.double(), groups, None, None, 1e-6, 1)
    d = group_norm_desc(L, x.shape, c, groups, 1e-6, 1, 1, 1)
    y = torch.empty_like(x)
    run_group_norm(L, d, x, None, None, y)
    check(y, want, size, HALF_STEP[torch.bfloat16])
    z = torch.empty_like(x)
    run_group_norm(L, d, x, None, None, z)
    assert torch.equal(y, z)
    run_group_norm(L, d, x, None, None, x)
    assert torch.equal(x, y)


@pytest.mark.parametrize("shape", [(1, 16, 16, 64, 8), (1, 128, 128, 256, 8), (1, 400, 300, 128, 4)],
                         ids=str)
def test_far_mean_and_constant_groups(shape):
    """A mean 1000 times the spread keeps its variance; a constant group gives
    beta, for eps alone."""
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c, groups = shape
    x, gamma, beta = inputs((n, h, w, c), 5, offset=0.0)
    x = x + 1000.0
    x[..., : c // groups] = 3.25
    d = group_norm_desc(L, x.shape, c, groups, 1e-5, 0, 0, 0)
    y = torch.empty_like(x)
    run_group_norm(L, d, x, gamma, beta, y)
    want, size = group_norm_64(x.double(), groups, gamma, beta, 1e-5, 0)
    check(y, want, size, HALF_STEP[torch.float32])


@pytest.mark.parametrize("act", range(5))
def test_non_finite_stays_in_its_group(act):
    import torch
    from computeengine_b200 import _lib as L
    x, gamma, beta = inputs((2, 20, 20, 64), 6)
    x[0, 3, 4, 17] = float("inf")
    x[1, 0, 0, 40] = float("nan")
    d = group_norm_desc(L, x.shape, 64, 8, 1e-5, act, 0, 0)
    y = torch.empty_like(x)
    run_group_norm(L, d, x, gamma, beta, y)
    bad = torch.isnan(y).all(dim=(1, 2))
    for n, g in ((0, 2), (1, 5)):
        assert bad[n, 8 * g:8 * g + 8].all()
        bad[n, 8 * g:8 * g + 8] = False
    assert not bad.any() and torch.isnan(y).sum() == 2 * 400 * 8


def test_extreme_activation_arguments():
    """SiLU and GELU far out: exactly z, or zero without NaN."""
    import torch
    from computeengine_b200 import _lib as L
    x = torch.randn(1, 8, 8, 32, device="cuda")
    gamma = torch.full((32,), 1e4, device="cuda")
    for act in (3, 4):
        y = torch.empty_like(x)
        run_group_norm(L, group_norm_desc(L, x.shape, 32, 4, 1e-5, act, 0, 0), x, gamma, None, y)
        want, size = group_norm_64(x.double(), 4, gamma, None, 1e-5, act)
        check(y, want, size, HALF_STEP[torch.float32])


def test_captured_and_replayed_on_another_stream():
    import torch
    from computeengine_b200 import _lib as L
    for shape in ((1, 8, 8, 64, 8), (1, 400, 300, 128, 4)):
        n, h, w, c, groups = shape
        x, gamma, beta = inputs((n, h, w, c), 7)
        y = torch.empty_like(x)
        d = group_norm_desc(L, x.shape, c, groups, 1e-5, 3, 0, 0)
        ws = torch.empty(max(int(L.lib.ie_cuda_group_norm_workspace_bytes(d)), 1),
                         dtype=torch.uint8, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            L.check(L.lib.ie_cuda_group_norm_nhwc(d, x.data_ptr(), gamma.data_ptr(),
                                                  beta.data_ptr(), y.data_ptr(), ws.data_ptr(),
                                                  ws.numel(),
                                                  torch.cuda.current_stream().cuda_stream))
        for k in range(3):
            x.mul_(1.5).add_(0.25 * k)
            g.replay()
            want, size = group_norm_64(x.double(), groups, gamma, beta, 1e-5, 3)
            check(y, want, size, HALF_STEP[torch.float32])


def test_more_than_32_bits_of_elements():
    """Offsets past 2^32 bytes and 2^31 elements: the last image equals the
    same image alone."""
    import torch
    from computeengine_b200 import _lib as L
    n, h, w, c = 17, 512, 512, 512
    one = inputs((1, h, w, c), 8)[0].bfloat16()
    x = torch.zeros(n, h, w, c, dtype=torch.bfloat16, device="cuda")
    x[-1] = one[0]
    run_group_norm(L, group_norm_desc(L, x.shape, c, 32, 1e-5, 3, 1, 1), x, None, None, x)
    y = torch.empty_like(one)
    run_group_norm(L, group_norm_desc(L, one.shape, c, 32, 1e-5, 3, 1, 1), one, None, None, y)
    assert torch.equal(x[-1], y[0])
    assert not x[:-1].any()


def test_operator():
    import torch
    from computeengine_b200.ops import Code, GroupNormOp
    x, gamma, beta = inputs((2, 12, 10, 48), 9)
    op = GroupNormOp()
    assert op.configure({"groups": 6, "activation": "SILU", "epsilon": 1e-6,
                         "dtype": torch.bfloat16})
    out = [None]
    view = x.permute(0, 2, 1, 3)  # strided
    st = op.forward([view, gamma, beta], out)
    assert st, st.message
    want, size = group_norm_64(view.double(), 6, gamma, beta, 1e-6, 3)
    check(out[0], want, size, HALF_STEP[torch.bfloat16])
    for bad, code in (([x.double()], Code.Unsupported), ([x[0]], Code.InvalidArgument),
                      ([x, gamma[:-1]], Code.InvalidArgument),
                      ([x[:0]], Code.InvalidArgument)):
        o = [None]
        st = op.forward(bad, o)
        assert not st and st.code == code and o == [None]
    assert op.configure({"groups": 7})
    assert op.forward([x], [None]).code == Code.InvalidArgument
