"""Attributes of the Python operators that the descriptors' types cannot hold are
refused with a status: none becomes another number, none raises."""
import math

import pytest


@pytest.mark.parametrize("op, attrs", [
    ("GroupNormOp", {"groups": (1 << 64) + 4}),
    ("GroupNormOp", {"groups": 4, "epsilon": 1e39}), ("GroupNormOp", {"groups": 4, "epsilon": 1e-60}),
    ("GroupNormOp", {"groups": 4, "epsilon": 10 ** 400}),
    ("GroupNormOp", {"groups": 4, "activation": ["SILU"]}),
    ("GroupNormOp", {"groups": 4, "dtype": {}}),
    ("RotaryOp", {"section": [(1 << 32) + 16]}), ("RotaryOp", {"section": [16, -(1 << 32) + 16]}),
    ("RotaryOp", {"section": [16], "rot_heads": (1 << 32) + 1}),
    ("RotaryOp", {"section": [16], "rot_heads": -(1 << 32) + 1}),
    ("RotaryOp", {"section": [16], "theta": 10 ** 400}),
    ("RotaryOp", {"section": [16], "layout": ["PAIRS"]}),
    ("AttentionOp", {"softcap": 1e-60}), ("AttentionOp", {"softcap": 1e39}),
    ("AttentionOp", {"scale": -1e39}), ("AttentionOp", {"scale": 1e-60}),
    ("AttentionOp", {"softcap": math.nan}), ("AttentionOp", {"softcap": 10 ** 400}),
])
def test_refused(op, attrs):
    from computeengine_b200 import ops
    st = getattr(ops, op)().configure(attrs)
    assert not st and st.code == ops.Code.InvalidArgument, st.message


@pytest.mark.parametrize("op, attrs", [
    ("GroupNormOp", {"groups": 4, "epsilon": 0}), ("GroupNormOp", {"groups": 4, "epsilon": 1e-40}),
    ("AttentionOp", {"softcap": 0}), ("AttentionOp", {"softcap": 3e38, "scale": 0.0}),
    ("AttentionOp", {"softcap": 1e-40}), ("RotaryOp", {"section": [16], "theta": 1e300}),
    ("RotaryOp", {"section": [0, 16], "rot_heads": 0}),
])
def test_taken(op, attrs):
    from computeengine_b200 import ops
    st = getattr(ops, op)().configure(attrs)
    assert st, st.message
