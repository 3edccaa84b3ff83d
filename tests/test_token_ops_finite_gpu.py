"""Group norm and attention over the sizes of their other tests, where a NaN is an
error: `not (error > tolerance).any()` lets one pass."""
import pytest

import tests.test_attention_gpu as attention
import tests.test_group_norm_gpu as group_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    within, check = attention.check_attention, group_norm.check

    def check_attention(o, lse, want, dtype, extra=0.0):
        assert not o[want[3]].isnan().any()
        within(o, lse, want, dtype, extra)

    def check_group_norm(y, want, size, half):
        assert not y.isnan().any()
        check(y, want, size, half)

    monkeypatch.setattr(attention, "check_attention", check_attention)
    monkeypatch.setattr(group_norm, "check", check_group_norm)


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("sq, sk", attention.LENGTHS, ids=str)
def test_attention_lengths(sq, sk, causal):
    attention.test_lengths(sq, sk, causal)


@pytest.mark.parametrize("dtype", attention.DTYPES)
@pytest.mark.parametrize("options", ["cap", "bias", "cap bias causal prefix", "prefix causal"])
@pytest.mark.parametrize("sq, sk, d", [(1, 333, 128), (9, 333, 80), (333, 333, 128), (260, 390, 64)],
                         ids=str)
def test_attention_scores_and_masks(sq, sk, d, options, dtype):
    attention.test_scores_and_masks(sq, sk, d, options, dtype)


@pytest.mark.parametrize("sq", [1, 3, 20, 150])
def test_attention_garbage_behind_lengths(sq):
    attention.test_ragged_lengths_with_garbage_behind_them(sq)


@pytest.mark.parametrize("sq", [1, 13, 200])
@pytest.mark.parametrize("d", [8, 72, 100])
def test_attention_head_dims(sq, d):
    attention.test_head_dims(sq, 150, d, "float16")


@pytest.mark.parametrize("shape", group_norm.SHAPES, ids=str)
@pytest.mark.parametrize("act", range(5))
def test_group_norm_shapes_and_activations(shape, act):
    group_norm.test_shapes_and_activations(shape, act)


@pytest.mark.parametrize("yt", group_norm.TYPES)
@pytest.mark.parametrize("xt", group_norm.TYPES)
@pytest.mark.parametrize("shape", [(2, 24, 24, 80, 96, 8), (1, 150, 160, 120, 128, 4)], ids=str)
def test_group_norm_types_and_padding_channels(shape, xt, yt):
    group_norm.test_types_and_padding_channels(shape, xt, yt)
