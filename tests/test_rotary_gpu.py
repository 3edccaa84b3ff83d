"""ie_cuda_rotary against the definition in 64 bits.

Tolerance: cos and sin in fp32 are off by at most two steps plus the rounding
of the angle to fp32 (half a step of at most half a turn: pi * 2^-24), the two
products and the sum by half a step each: below 8 half steps of |u| + |v|; then
one rounding to the output type.  Below 2^-14 the steps of fp16 stay 2^-24, so
that rounding is off by up to 2^-25 however small the value is, which half a
step relative to the value does not cover: a copied x = 1.5 * 2^-24 lies half
way between two fp16 numbers and is off by 2^-25, where 2^-11 x + 2^-21 x is
below 2^-34.  (fp32 and bf16 reach down to 2^-126.)  The 64-bit angles are themselves off by
position * 2^-53, the fixed-point ones by position * 2^-65 turns: nothing at
the positions used."""
import pytest

from tests.token_ops import HALF_STEP, rotary_64, rotary_desc, rotary_pairs, run_rotary

pytestmark = pytest.mark.gpu


def check(y, want, size, dtype):
    import torch
    err = (y.double() - want).abs()
    tol = HALF_STEP[dtype] * want.abs() + 8 * 2.0 ** -24 * size + 2.0 ** -25 * size.clamp(max=1)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert not (err > tol).any(), float((err / tol.clamp(min=1e-30)).max())
    assert not torch.isnan(y).any()


def positions(axes, tokens, far, bits=32, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.randint(-3, far + 1, (axes, tokens), generator=g, device="cuda")
    return p.to(torch.int64 if bits == 64 else torch.int32)


# head_dim, section: vectors that fit, sections that end inside one, odd
# numbers of pairs, pass-through elements, one pair, an empty section
HEADS = [(128, (16, 24, 24)), (64, (16, 16)), (72, (18, 18)), (128, (22, 21, 21)), (32, (16,)),
         (96, (8, 8)), (80, (10, 20, 5)), (2, (1,)), (5, (1, 1)), (256, (32, 32, 32, 32)),
         (64, (0, 32)), (66, (11, 11, 11)), (40, (3,))]


@pytest.mark.parametrize("freq", [0, 1])
@pytest.mark.parametrize("layout", [0, 1, 2])
@pytest.mark.parametrize("head", HEADS, ids=str)
def test_layouts(head, layout, freq):
    import torch
    from computeengine_b200 import _lib as L
    d, section = head
    x = torch.randn(37, 5, d, device="cuda")
    y = torch.full_like(x, float("nan"))
    pos = positions(len(section), 37, 5000)
    run_rotary(L, rotary_desc(L, x, y, 3, section, layout, freq, pos), x, pos, y)
    check(y, *rotary_64(x, pos, 3, section, layout, freq), torch.float32)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("yt", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("xt", ["float32", "bfloat16", "float16"])
def test_types(xt, yt, bits):
    import torch
    from computeengine_b200 import _lib as L
    for d, section in ((128, (16, 24, 24)), (72, (18, 18)), (30, (7, 4))):
        x = torch.randn(11, 7, d, device="cuda").to(getattr(torch, xt))
        y = torch.full(x.shape, float("nan"), dtype=getattr(torch, yt), device="cuda")
        pos = positions(len(section), 11, 70000, bits)
        run_rotary(L, rotary_desc(L, x, y, 4, section, 1, 0, pos), x, pos, y)
        check(y, *rotary_64(x, pos, 4, section, 1, 0), y.dtype)


@pytest.mark.parametrize("tokens", [1, 2, 8, 257, 5000])
@pytest.mark.parametrize("heads", [1, 40])
def test_token_counts(tokens, heads):
    import torch
    from computeengine_b200 import _lib as L
    x = torch.randn(tokens, heads, 128, device="cuda").bfloat16()
    y = torch.full_like(x, float("nan"))
    pos = positions(3, tokens, 1000000)
    run_rotary(L, rotary_desc(L, x, y, heads, (16, 24, 24), 1, 0, pos), x, pos, y)
    check(y, *rotary_64(x, pos, heads, (16, 24, 24), 1, 0), torch.bfloat16)


def test_far_positions_and_inverse():
    """Positions up to 2^24 (64-bit angles are off by 2^-29 there); the inverse
    brings x back to two roundings."""
    import torch
    from computeengine_b200 import _lib as L
    x = torch.randn(200, 2, 64, device="cuda")
    pos = positions(1, 200, 1 << 24)
    y, z = torch.empty_like(x), torch.empty_like(x)
    run_rotary(L, rotary_desc(L, x, y, 2, (32,), 0, 0, pos), x, pos, y)
    check(y, *rotary_64(x, pos, 2, (32,), 0, 0), torch.float32)
    run_rotary(L, rotary_desc(L, y, z, 2, (32,), 0, 0, pos, inverse=1), y, pos, z)
    check(z, *rotary_64(y, pos, 2, (32,), 0, 0, inverse=1), torch.float32)
    assert float((z - x).abs().max()) < 1e-5


def test_whole_turns_of_64_bit_positions():
    """theta = 1 rotates by the position itself, in radians; 64-bit positions
    are taken whole: 2^40 + p against the angle in extended precision."""
    import numpy as np
    import torch
    from computeengine_b200 import _lib as L
    p = (1 << 36) + np.arange(50, dtype=np.int64)
    pos = torch.from_numpy(p).cuda()[None]
    x = torch.tensor([1.0, 0.0], device="cuda").expand(50, 1, 2).contiguous()
    y = torch.empty_like(x)
    run_rotary(L, rotary_desc(L, x, y, 1, (1,), 0, 0, pos, theta=1.0), x, pos, y)
    # 2^36 / (2 pi) turns: 2^-65 turns off per position, 2^-29 turns in all;
    # the same in long double is off by 2^36 * 2^-64
    two_pi = np.longdouble("6.283185307179586476925286766559")
    r = np.fmod(p.astype(np.longdouble), two_pi)
    tol = 2 * np.pi * 2.0 ** -29 + 8 * 2.0 ** -24
    assert np.abs(y[:, 0, 0].cpu().numpy() - np.cos(r).astype(np.float64)).max() < tol
    assert np.abs(y[:, 0, 1].cpu().numpy() - np.sin(r).astype(np.float64)).max() < tol


@pytest.mark.parametrize("d, section, layout", [(128, (16, 24, 24), 1), (64, (16, 8), 0),
                                                (72, (18, 18), 2), (36, (9, 9), 1)])
def test_strides_in_place_and_neighbours(d, section, layout):
    """q and k inside packed qkv rows, rotated in place; all else untouched."""
    import torch
    from computeengine_b200 import _lib as L
    rows = torch.randn(65, 3 * 4 * d + 24, device="cuda").bfloat16()
    before = rows.clone()
    x = rows[:, 8:8 + 8 * d].view(65, 8, d)
    pos = positions(len(section), 65, 4000)
    want, size = rotary_64(x, pos, 8, section, layout, 1)
    run_rotary(L, rotary_desc(L, x, x, 8, section, layout, 1, pos), x, pos, x)
    check(x, want, size, torch.bfloat16)
    rest = rows.clone()
    rest[:, 8:8 + 8 * d] = before[:, 8:8 + 8 * d]
    assert torch.equal(rest, before)
    used = {e for _, _, u, v in rotary_pairs(section, layout, 1, 1e4) for e in (u, v)}
    for e in set(range(d)) - used:
        assert torch.equal(x[..., e], before[:, 8:8 + 8 * d].view(65, 8, d)[..., e])


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_orders_and_alignment(shift):
    """Heads outermost, odd row strides, pointers off every vector boundary."""
    import torch
    from computeengine_b200 import _lib as L
    d, section, tokens, heads = 64, (10, 22), 19, 6
    for dt in (torch.float32, torch.bfloat16):
        x = torch.randn(heads, tokens, d + 3, device="cuda").to(dt)[:, :, shift:shift + d]
        x = x.transpose(0, 1)
        y = torch.full((heads, tokens, d + 5), 7.0, device="cuda", dtype=dt)
        yv = y[:, :, shift:shift + d].transpose(0, 1)
        pos = positions(4, tokens, 300)[::2]  # an axis stride
        run_rotary(L, rotary_desc(L, x, yv, 4, section, 1, 0, pos), x, pos, yv)
        check(yv, *rotary_64(x, pos, 4, section, 1, 0), dt)
        assert (y[:, :, :shift] == 7).all() and (y[:, :, shift + d:] == 7).all()


def test_broadcast_x():
    """One token's x at many positions (token stride 0)."""
    import torch
    from computeengine_b200 import _lib as L
    x = torch.randn(1, 4, 64, device="cuda").expand(50, 4, 64)
    y = torch.empty(50, 4, 64, device="cuda")
    pos = positions(2, 50, 900)
    run_rotary(L, rotary_desc(L, x, y, 4, (16, 16), 1, 0, pos), x, pos, y)
    check(y, *rotary_64(x, pos, 4, (16, 16), 1, 0), torch.float32)


def test_more_than_32_bits_of_elements():
    import torch
    from computeengine_b200 import _lib as L
    tokens, heads, d = 70000, 256, 128
    x = torch.zeros(tokens, heads, d, dtype=torch.bfloat16, device="cuda")
    x[-9:] = torch.randn(9, heads, d, device="cuda").bfloat16()
    pos = positions(1, tokens, 9000)
    tail, tpos = x[-9:].clone(), pos[:, -9:].contiguous()
    run_rotary(L, rotary_desc(L, x, x, heads, (64,), 1, 0, pos), x, pos, x)
    y = torch.empty_like(tail)
    run_rotary(L, rotary_desc(L, tail, y, heads, (64,), 1, 0, tpos), tail, tpos, y)
    assert torch.equal(x[-9:], y) and not x[:-9].any()


def test_gradient_is_the_inverse():
    """<g, R x> = <R^-1 g, x>, and differences of a loss along x."""
    import torch
    from computeengine_b200 import _lib as L
    x, g = torch.randn(2, 9, 3, 64, device="cuda").double().float()
    pos = positions(2, 9, 500)
    y, gx = torch.empty_like(x), torch.empty_like(x)
    run_rotary(L, rotary_desc(L, x, y, 3, (20, 12), 1, 1, pos), x, pos, y)
    run_rotary(L, rotary_desc(L, x, gx, 3, (20, 12), 1, 1, pos, inverse=1), g, pos, gx)
    a, b = (g.double() * y.double()).sum(), (gx.double() * x.double()).sum()
    # each of the 1728 products is off by at most 9 half steps of about its size
    scale = float((g.double().norm() * x.double().norm()))
    assert abs(float(a - b)) <= 2 * 9 * 2.0 ** -24 * scale * 2
    h, e = 2.0 ** -4, torch.randn_like(x)
    yp = torch.empty_like(x)
    xp = x + h * e
    run_rotary(L, rotary_desc(L, xp, yp, 3, (20, 12), 1, 1, pos), xp, pos, yp)
    slope = float(((yp.double() - y.double()) * g.double()).sum()) / h
    want = float((gx.double() * (xp.double() - x.double())).sum()) / h
    assert abs(slope - want) <= 2 * 9 * 2.0 ** -24 * scale / h * 4


def test_captured_and_replayed():
    import torch
    from computeengine_b200 import _lib as L
    x = torch.randn(8, 40, 128, device="cuda").bfloat16()
    y = torch.empty_like(x)
    pos = positions(3, 8, 1000)
    d, plan = rotary_desc(L, x, y, 40, (16, 24, 24), 1, 0, pos), L.RotaryPlan()
    L.check(L.lib.ie_rotary_plan_init(d, plan))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.check(L.lib.ie_cuda_rotary(d, plan, x.data_ptr(), pos.data_ptr(), y.data_ptr(),
                                     torch.cuda.current_stream().cuda_stream))
    del plan, d  # a captured launch holds its own copy
    for step in range(3):
        pos.add_(1)
        g.replay()
        check(y, *rotary_64(x, pos, 40, (16, 24, 24), 1, 0), torch.bfloat16)


def test_operator():
    import torch
    from computeengine_b200.ops import Code, RotaryOp
    x = torch.randn(30, 6, 72, device="cuda")
    pos = positions(2, 30, 100, 64)
    op = RotaryOp()
    assert op.configure({"section": [18, 18], "layout": "AXIS_HALVES", "frequencies": "PER_AXIS",
                         "rot_heads": 4, "dtype": torch.bfloat16})
    out = [None]
    st = op.forward([x, pos], out)
    assert st, st.message
    check(out[0], *rotary_64(x, pos, 4, (18, 18), 2, 1), torch.bfloat16)
    for bad, code in (([x, pos[:1]], Code.InvalidArgument), ([x[0], pos], Code.InvalidArgument),
                      ([x.double(), pos], Code.Unsupported), ([x, pos.float()], Code.Unsupported),
                      ([x[..., :30], pos], Code.InvalidArgument)):
        o = [None]
        st = op.forward(bad, o)
        assert not st and st.code == code and o == [None]
