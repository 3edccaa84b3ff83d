"""Rotary positions and attention refuse outputs whose rows share elements, by any
two of their strides, before any CUDA call."""
import pytest

from tests.test_token_ops_cpu import FAKE, _att, _lib, _rot


@pytest.mark.parametrize("kw", [
    dict(y_token_stride=64, y_head_stride=64),    # tokens over heads
    dict(y_token_stride=128, y_head_stride=64),   # heads 2 and 3 over the next token
    dict(y_token_stride=64, y_head_stride=192),   # tokens 3 over the next head
    dict(y_token_stride=1 << 62, y_head_stride=1 << 62, tokens=8),  # behind the last address
])
def test_rotary(kw):
    L = _lib()
    plan = L.RotaryPlan()
    d = _rot(L, **kw)
    assert L.lib.ie_rotary_plan_init(d, plan) == 0
    assert L.lib.ie_cuda_rotary(d, plan, FAKE, FAKE, 2 * FAKE, None) == L.IE_INVALID_ARGUMENT
    assert b"overlap" in L.lib.ie_cuda_last_error()


@pytest.mark.parametrize("kw", [  # batch 2, 8 positions, 4 heads of 64
    dict(o_stride=(2048, 64, 64)), dict(o_stride=(2048, 128, 64)), dict(o_stride=(64, 256, 64)),
    dict(o_stride=(1024, 256, 64)), dict(o_stride=(2048, 64, 448)),
    dict(o_stride=(1 << 62, 1 << 61, 64)),
    # split: the lo planes over other heads' hi planes, other tokens or rows of the batch
    dict(o_type=3, o_stride=(4096, 256, 64)), dict(o_type=3, o_stride=(4096, 510, 64)),
    dict(o_type=3, o_stride=(2048, 512, 64)), dict(o_type=3, o_stride=(2048, 128, 512)),
])
def test_attention(kw):
    L = _lib()
    d = _att(L, **kw)
    rc = L.lib.ie_cuda_attention(d, None, FAKE, FAKE, FAKE, FAKE, None, FAKE, 1 << 30, None)
    assert rc == L.IE_INVALID_ARGUMENT and b"overlap" in L.lib.ie_cuda_last_error()
    assert L.lib.ie_cuda_attention_workspace_bytes(d, None) == 0


def test_attention_split_planes_of_a_single_position():
    """The token stride places the lo plane even where there is one token."""
    L = _lib()
    d = _att(L, batch=1, q_len=1, o_type=3, o_stride=(0, 256, 64))
    assert L.lib.ie_cuda_attention(d, None, FAKE, FAKE, FAKE, FAKE, None, FAKE, 1 << 30,
                                   None) == L.IE_INVALID_ARGUMENT
