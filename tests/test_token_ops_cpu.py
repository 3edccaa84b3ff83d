"""Group norm, rotary positions and attention without a GPU: every refusal of
the C ABI comes before any CUDA call, and the rotary plan's frequencies."""
import math

import numpy as np
import pytest


def _lib():
    from computeengine_b200 import _lib as L
    return L


FAKE = 0x1000  # never read: the calls below are refused first


def _gn(L, **kw):
    base = dict(n=1, c=64, h=4, w=4, c_store=64, groups=8, eps=1e-5, act=0, x_type=0, y_type=0)
    base.update(kw)
    return L.GroupNormDesc(**base)


@pytest.mark.parametrize("kw, code", [
    (dict(n=0), 1), (dict(c=0), 1), (dict(h=-1), 1), (dict(w=0), 1), (dict(groups=0), 1),
    (dict(groups=7), 1), (dict(c_store=63), 1), (dict(eps=-1.0), 1), (dict(eps=math.nan), 1),
    (dict(eps=math.inf), 1), (dict(act=5), 1), (dict(act=-1), 1), (dict(x_type=4), 1),
    (dict(y_type=-1), 1), (dict(c_store=72, y_type=3), 1), (dict(c_store=72, x_type=3), 1),
    (dict(h=1 << 20, w=1 << 20), 2), (dict(n=1 << 16), 2),
    (dict(h=(1 << 62), w=4), 2),
    (dict(c=1 << 21, c_store=1 << 21), 2),
])
def test_group_norm_refusals(kw, code):
    L = _lib()
    assert L.lib.ie_cuda_group_norm_nhwc(_gn(L, **kw), FAKE, None, None, FAKE, None, 0,
                                         None) == code
    assert L.lib.ie_cuda_last_error()
    assert L.lib.ie_cuda_group_norm_workspace_bytes(_gn(L, **kw)) == 0


def test_group_norm_refuses_null_and_mixed_in_place():
    L = _lib()
    f = L.lib.ie_cuda_group_norm_nhwc
    assert f(None, FAKE, None, None, FAKE, None, 0, None) == L.IE_INVALID_ARGUMENT
    assert f(_gn(L), None, None, None, FAKE, None, 0, None) == L.IE_INVALID_ARGUMENT
    assert f(_gn(L), FAKE, None, None, None, None, 0, None) == L.IE_INVALID_ARGUMENT
    assert f(_gn(L, y_type=1), FAKE, None, None, FAKE, None, 0, None) == L.IE_INVALID_ARGUMENT


def test_convolutions_refuse_the_group_norm_activations():
    L = _lib()
    from tests.qconv import desc_for
    d = desc_for(L, 1, 16, 8, 8, 16, 3, 3, (1, 1), (1, 1, 1, 1))
    for act in (L.IE_ACT_SILU, L.IE_ACT_GELU):
        assert L.lib.ie_cuda_conv2d_f32(d, act, FAKE, FAKE, None, FAKE, FAKE, 1 << 30,
                                        None) == L.IE_INVALID_ARGUMENT


def _rot(L, section=(16, 16), **kw):
    base = dict(tokens=4, x_token_stride=256, x_head_stride=64, y_token_stride=256,
                y_head_stride=64, pos_axis_stride=4, theta=10000.0, heads=4, rot_heads=4,
                head_dim=64, axes=len(section), layout=1, freq=0, inverse=0, x_type=0, y_type=0,
                pos_bits=32)
    base.update(kw)
    d = L.RotaryDesc(**base)
    for i, s in enumerate(section[:4]):
        d.section[i] = s
    return d


@pytest.mark.parametrize("section, kw, code", [
    ((16, 16), dict(head_dim=0), 1), ((16, 16), dict(head_dim=257), 2), ((16, 17), {}, 1),
    ((0, 0), {}, 1), ((33, -1), {}, 1), ((16, 16), dict(axes=0), 1), ((16, 16), dict(axes=5), 1),
    ((16, 16), dict(layout=3), 1), ((16, 16), dict(freq=2), 1), ((16, 16), dict(theta=0.0), 1),
    ((16, 16), dict(theta=math.inf), 1), ((16, 16), dict(theta=math.nan), 1),
])
def test_rotary_plan_refusals(section, kw, code):
    L = _lib()
    assert L.lib.ie_rotary_plan_init(_rot(L, section, **kw), L.RotaryPlan()) == code


@pytest.mark.parametrize("kw, code", [
    (dict(tokens=0), 1), (dict(heads=0), 1), (dict(rot_heads=5), 1), (dict(rot_heads=-1), 1),
    (dict(x_type=3), 1), (dict(y_type=3), 1), (dict(pos_bits=16), 1),
    (dict(x_token_stride=-1), 1), (dict(y_head_stride=32), 1), (dict(y_token_stride=0), 1),
    (dict(pos_axis_stride=-4), 1), (dict(tokens=1 << 31), 2), (dict(theta=500.0), 1),
    (dict(layout=0), 1), (dict(freq=1), 1), (dict(head_dim=72), 1),
])
def test_rotary_refusals(kw, code):
    L = _lib()
    plan = L.RotaryPlan()
    assert L.lib.ie_rotary_plan_init(_rot(L), plan) == 0
    assert L.lib.ie_cuda_rotary(_rot(L, **kw), plan, FAKE, FAKE, 2 * FAKE, None) == code


def test_rotary_refuses_null_and_mixed_in_place():
    L = _lib()
    plan = L.RotaryPlan()
    assert L.lib.ie_rotary_plan_init(_rot(L), None) == L.IE_INVALID_ARGUMENT
    assert L.lib.ie_rotary_plan_init(_rot(L), plan) == 0
    f = L.lib.ie_cuda_rotary
    for args in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None)):
        assert f(_rot(L), plan, *args, None) == L.IE_INVALID_ARGUMENT
    assert f(_rot(L), None, FAKE, FAKE, FAKE, None) == L.IE_INVALID_ARGUMENT
    assert f(_rot(L, y_type=1), plan, FAKE, FAKE, FAKE, None) == L.IE_INVALID_ARGUMENT
    assert f(_rot(L, y_token_stride=512), plan, FAKE, FAKE, FAKE, None) == L.IE_INVALID_ARGUMENT


def test_rotary_plan_frequencies():
    """turns / 2^64 is the frequency over 2 pi: half a step of the fixed point is
    2^-65 absolute, and 2 * math.pi is pi rounded to 53 bits, 2^-53 relative."""
    L = _lib()
    for section, freq in (((10, 6, 16), 0), ((10, 6, 16), 1), ((32,), 0)):
        plan = L.RotaryPlan()
        assert L.lib.ie_rotary_plan_init(_rot(L, section, freq=freq, axes=len(section)), plan) == 0
        i = 0
        for a, size in enumerate(section):
            for j in range(size):
                e = np.longdouble(i) / 32 if freq == 0 else np.longdouble(j) / size
                f = np.longdouble(10000.0) ** -e / (2 * np.longdouble(math.pi))
                tol = 2.0 ** -52 * float(f) + 2.0 ** -64
                assert abs(float(plan.turns[i]) * 2.0 ** -64 - float(f)) <= tol
                assert plan.axis[i] == a
                i += 1
        assert plan.pairs == 32


def _att(L, **kw):
    strides = {k: kw.pop(k) for k in list(kw) if k.endswith("stride")}
    base = dict(batch=2, q_len=8, kv_len=8, q_heads=4, kv_heads=2, head_dim=64, type=1, o_type=1,
                scale=0.125, softcap=0.0)
    base.update(kw)
    d = L.AttentionDesc(**base)
    for name, heads in (("q", 4), ("k", 2), ("v", 2), ("o", 4)):
        for i, s in enumerate(strides.get(name + "_stride", (8 * heads * 64, heads * 64, 64))):
            getattr(d, name + "_stride")[i] = s
    return d


@pytest.mark.parametrize("kw, code", [
    (dict(batch=0), 1), (dict(q_len=0), 1), (dict(kv_len=0), 1), (dict(q_heads=0), 1),
    (dict(kv_heads=0), 1), (dict(kv_heads=3), 1), (dict(head_dim=0), 1), (dict(head_dim=129), 2),
    (dict(type=0, o_type=0), 2), (dict(type=3, o_type=3), 2), (dict(type=7), 1),
    (dict(o_type=2), 1), (dict(type=2, o_type=3), 1), (dict(o_type=0), 1),
    (dict(scale=math.nan), 1), (dict(scale=math.inf), 1), (dict(softcap=-1.0), 1),
    (dict(softcap=math.nan), 1), (dict(softcap=math.inf), 1), (dict(batch=1 << 16), 2),
    (dict(q_len=(1 << 30) + 1), 2), (dict(kv_len=1 << 40), 2),
    (dict(q_stride=(-1, 256, 64)), 1), (dict(o_stride=(2048, 256, 32)), 1),
    (dict(o_stride=(0, 256, 64)), 1), (dict(o_type=3, o_stride=(2048, 64, 1024)), 1),
])
def test_attention_refusals(kw, code):
    L = _lib()
    d = _att(L, **kw)
    assert L.lib.ie_cuda_attention(d, None, FAKE, FAKE, FAKE, FAKE, None, None, 0, None) == code
    assert L.lib.ie_cuda_attention_workspace_bytes(d, None) == 0


@pytest.mark.parametrize("batch, kw", [
    (2, dict(documents=-1)),
    (2, dict(documents=2, q_offsets=FAKE, kv_offsets=FAKE)),
    (1, dict(documents=2, q_offsets=FAKE)),
    (1, dict(documents=2, kv_offsets=FAKE)),
    (1, dict(documents=2, q_offsets=FAKE, kv_offsets=FAKE, kv_lens=FAKE)),
    (2, dict(prefix_lens=FAKE)),
])
def test_attention_mask_refusals(batch, kw):
    L = _lib()
    rc = L.lib.ie_cuda_attention(_att(L, batch=batch), L.AttentionMask(**kw), FAKE, FAKE, FAKE,
                                 FAKE, None, None, 0, None)
    assert rc == L.IE_INVALID_ARGUMENT


def test_attention_refuses_null_tensors():
    L = _lib()
    for i in range(4):
        args = [FAKE] * 4
        args[i] = None
        assert L.lib.ie_cuda_attention(_att(L), None, *args, None, None, 0,
                                       None) == L.IE_INVALID_ARGUMENT
    assert L.lib.ie_cuda_attention(None, None, FAKE, FAKE, FAKE, FAKE, None, None, 0,
                                   None) == L.IE_INVALID_ARGUMENT


def test_ops_configure_refusals():
    """The Python operators check their attributes like the convolution ops."""
    from computeengine_b200.ops import AttentionOp, Code, GroupNormOp, OpRegistry, RotaryOp
    from computeengine_b200.ops import register_cuda_ops
    reg = OpRegistry()
    assert register_cuda_ops(reg)
    for name, cls in (("GroupNorm", GroupNormOp), ("Rotary", RotaryOp), ("Attention", AttentionOp)):
        op, st = reg.create(name)
        assert st and isinstance(op, cls)
    for cls, attrs in ((GroupNormOp, {}), (GroupNormOp, {"groups": 0}),
                       (GroupNormOp, {"groups": 4, "epsilon": -1.0}),
                       (GroupNormOp, {"groups": 4, "activation": "TANH"}),
                       (RotaryOp, {}), (RotaryOp, {"section": []}),
                       (RotaryOp, {"section": [1, 2, 3, 4, 5]}),
                       (RotaryOp, {"section": [4], "layout": "ROWS"}),
                       (RotaryOp, {"section": [4], "frequencies": "NONE"}),
                       (AttentionOp, {"softcap": -1.0}), (AttentionOp, {"causal": "yes"}),
                       (AttentionOp, {"scale": math.inf})):
        st = cls().configure(attrs)
        assert not st and st.code == Code.InvalidArgument, (cls, attrs)


def test_ops_refuse_host_tensors():
    import torch
    from computeengine_b200.ops import AttentionOp, Code, GroupNormOp, RotaryOp
    x = torch.zeros(1, 4, 4, 16)
    for op, attrs, inputs in (
            (GroupNormOp(), {"groups": 4}, [x]),
            (RotaryOp(), {"section": [4]}, [x[0], torch.zeros(1, 4, dtype=torch.int32)]),
            (AttentionOp(), {}, [x.bfloat16()] * 3)):
        assert op.configure(attrs)
        out = [None]
        st = op.forward(inputs, out)
        assert not st and st.code == Code.InvalidArgument and out == [None]
