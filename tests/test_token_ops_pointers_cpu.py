"""Group norm, rotary positions and attention refuse pointers that are not aligned
to their elements (a GPU cannot read such an element) before any CUDA call."""
import pytest

from tests.test_token_ops_cpu import FAKE, _att, _gn, _lib, _rot


def _refused(L, rc):
    return rc == L.IE_INVALID_ARGUMENT and b"aligned" in L.lib.ie_cuda_last_error()


@pytest.mark.parametrize("types", [(0, 0), (1, 1), (2, 0), (0, 3), (3, 3)])
def test_group_norm(types):
    L = _lib()
    x_bytes, y_bytes = (4 if t == 0 else 2 for t in types)
    d = _gn(L, x_type=types[0], y_type=types[1])
    good = [FAKE, FAKE, FAKE, 2 * FAKE]
    for at, step in ((0, x_bytes), (1, 4), (2, 4), (3, y_bytes)):
        for off in range(1, step):
            p = list(good)
            p[at] += off
            rc = L.lib.ie_cuda_group_norm_nhwc(d, p[0], p[1], p[2], p[3], FAKE, 1 << 20, None)
            assert _refused(L, rc), (at, off)


@pytest.mark.parametrize("x_type, y_type, bits", [(0, 0, 32), (1, 1, 64), (0, 2, 64), (2, 0, 32)])
def test_rotary(x_type, y_type, bits):
    L = _lib()
    plan = L.RotaryPlan()
    d = _rot(L, x_type=x_type, y_type=y_type, pos_bits=bits)
    assert L.lib.ie_rotary_plan_init(d, plan) == 0
    for at, step in ((0, 4 if x_type == 0 else 2), (1, bits // 8), (2, 4 if y_type == 0 else 2)):
        for off in range(1, step):
            p = [FAKE, FAKE, 2 * FAKE]
            p[at] += off
            assert _refused(L, L.lib.ie_cuda_rotary(d, plan, *p, None)), (at, off)


@pytest.mark.parametrize("dtype", [1, 2])
def test_attention(dtype):
    L = _lib()
    d = _att(L, batch=1, type=dtype, o_type=dtype)

    def call(tensors=(FAKE,) * 4, lse=None, **mask):
        m = L.AttentionMask(**mask)
        return L.lib.ie_cuda_attention(d, m, *tensors, lse, FAKE, 1 << 30, None)

    for at in range(4):
        p = [FAKE] * 4
        p[at] += 1
        assert _refused(L, call(p)), at
    for off in (1, 2, 3):
        assert _refused(L, call(lse=FAKE + off))
        assert _refused(L, call(kv_lens=FAKE + off))
        assert _refused(L, call(causal=1, prefix_lens=FAKE + off))
        assert _refused(L, call(slopes=FAKE + off))
        assert _refused(L, call(documents=1, q_offsets=FAKE + off, kv_offsets=FAKE))
        assert _refused(L, call(documents=1, q_offsets=FAKE, kv_offsets=FAKE + off))
