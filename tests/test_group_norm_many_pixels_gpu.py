"""Group normalization of an image of very many pixels: a thread adds thousands of equal
squares, each of which the sum would round the same way."""
import pytest

from tests.token_ops import group_norm_desc, run_group_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h, c, value", [(1024, 2048, 0.3169), (512, 2040, 0.7071)])
def test_two_values(h, c, value):
    """Half of the pixels hold `value`, the others its negative: y is value / sigma up to
    72 half steps of twice that (the constant of test_group_norm_gpu.py)."""
    import torch
    from computeengine_b200 import _lib as L
    v = torch.tensor(value).bfloat16().item()
    x = torch.full((1, h, 1024, c), v, dtype=torch.bfloat16, device="cuda")
    x[:, :, ::2] = -v
    y = torch.empty(x.shape, device="cuda")
    run_group_norm(L, group_norm_desc(L, x.shape, c, 8, 1e-5, 0, 1, 0), x, None, None, y)
    want = v / (v * v + 1e-5) ** 0.5
    tol = 2 * 72 * 2.0 ** -24 * want
    assert (y[:, :, 1::2] - want).abs().max() <= tol
    assert (y[:, :, ::2] + want).abs().max() <= tol
