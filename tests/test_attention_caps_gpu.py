"""Attention's tanh cap over every size that the descriptor takes, in the kernel
for few rows (one query) and the one for many."""
import pytest

from tests.test_attention_gpu import ints, run_and_check as run_and_compare, tensors
from tests.token_ops import (attention_64, attention_desc, attention_mask, check_attention,
                             run_attention)

pytestmark = pytest.mark.gpu


def run_and_check(*tensors, **options):
    """Nor may any output be NaN, which compares as within a tolerance."""
    o, _, _ = run_and_compare(*tensors, **options)
    assert not o.isnan().any()


@pytest.mark.parametrize("sq", [1, 3, 40, 130])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e9, 1e20, 3e38])
def test_large_caps_leave_ordinary_scores(cap, dtype, sq):
    for d, gain in ((64, 0.5), (128, 4.0)):
        run_and_check(*tensors(2, sq, 300, 4, 2, d, dtype, seed=7, gain=gain), softcap=cap,
                      causal=int(sq > 1))


@pytest.mark.parametrize("sq", [1, 130])
@pytest.mark.parametrize("cap", [1e-3, 1e-20, 1e-37, 1e-40])
def test_tiny_caps_make_all_keys_equal(cap, sq):
    q, k, v = tensors(2, sq, 300, 4, 2, 64, seed=8)
    q[:, :, 0] = 0  # scores of exactly zero
    run_and_check(q, k, v, softcap=cap)


@pytest.mark.parametrize("sq", [1, 9, 130])
@pytest.mark.parametrize("cap", [1e5, 1e7])
def test_large_caps_beside_garbage(cap, sq):
    """Keys behind the sequences' lengths hold NaN, infinities and large numbers."""
    q, k, v = tensors(3, sq, 200, 4, 2, 128, seed=9)
    lens = ints(150, 129, 7)
    for n, l in enumerate(lens.tolist()):
        k[n, l:] = (float("nan"), float("inf"), 3e38)[n]
        v[n, l:] = float("nan")
    run_and_check(q, k, v, softcap=cap, kv_lens=lens)


@pytest.mark.parametrize("sq", [8, 130])
@pytest.mark.parametrize("cap", [1e5, 1e6])
def test_small_scores_beside_large_ones(cap, sq):
    """Every other query's scores reach the cap; the others' stay what they are."""
    import torch
    from computeengine_b200 import _lib as L
    q, k, v = tensors(1, sq, 300, 2, 2, 64, seed=10)
    q[:, 1::2] *= 1e7
    o, lse = torch.empty_like(q), torch.empty(1, 2, sq, device="cuda")
    run_attention(L, attention_desc(L, q, k, v, o, 0.125, cap), attention_mask(L), q, k, v, o, lse)
    want = attention_64(q, k, v, 0.125, cap)
    rows = want[3].clone()
    rows[:, 1::2] = False
    check_attention(o, lse, (*want[:3], rows), q.dtype)
    assert not torch.isnan(o).any() and not torch.isnan(lse).any()
