"""The operators on tensors of a device that is not the current one, and on a
side stream."""
import pytest

from tests.token_ops import attention_64, check_attention, group_norm_64, rotary_64

pytestmark = pytest.mark.gpu


def run_all(device):
    import torch
    from computeengine_b200.ops import AttentionOp, GroupNormOp, RotaryOp
    g = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(2, 20, 20, 64, generator=g, device=device)
    gn, rot, att = GroupNormOp(), RotaryOp(), AttentionOp()
    assert gn.configure({"groups": 8, "activation": "SILU"})
    assert rot.configure({"section": [8, 8], "dtype": torch.bfloat16})
    assert att.configure({"causal": True})
    out = [None]
    assert gn.forward([x], out)
    y = out[0]
    pos = torch.arange(800, device=device).repeat(2, 1)
    assert rot.forward([y.view(800, 2, 32), pos], out)
    q = out[0].view(2, 400, 2, 32)
    r = out[0]
    assert att.forward([q, q, q], out)
    torch.cuda.synchronize(device)
    want, size = group_norm_64(x.double(), 8, None, None, 1e-5, 3)
    assert not ((y.double() - want).abs() > 2.0 ** -17 * (size + 1)).any()
    want, size = rotary_64(y.view(800, 2, 32), pos, 2, (8, 8), 1, 0)
    assert not ((r.double() - want).abs() > 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).any()
    check_attention(out[0], None, attention_64(q, q, q, 32 ** -0.5, causal=1), torch.bfloat16)


def test_side_stream():
    import torch
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run_all("cuda:0")


def test_device_that_is_not_current():
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two visible GPUs")
    assert torch.cuda.current_device() == 0
    run_all("cuda:1")


def test_tensors_of_several_devices_are_refused():
    import torch
    from computeengine_b200.ops import Code, GroupNormOp
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two visible GPUs")
    op, out = GroupNormOp(), [None]
    assert op.configure({"groups": 4})
    st = op.forward([torch.zeros(1, 2, 2, 16, device="cuda:0"), torch.ones(16, device="cuda:1")],
                    out)
    assert not st and st.code == Code.InvalidArgument
