"""A block of a network that mixes convolutions with attention, run through the
C ABI end to end: x -> group norm + SiLU -> 1x1 convolution (q, k, v) -> rotary
positions by height and width -> attention -> 1x1 convolution + x, all channels
last, each step reading what the step before wrote."""
import pytest

from tests.token_ops import (attention_64, attention_desc, attention_mask, group_norm_64,
                             group_norm_desc, joined, rotary_64, rotary_desc, run_attention,
                             run_group_norm, run_rotary, stream)

pytestmark = pytest.mark.gpu


def conv_desc(n, h, w, cin, cout):
    from computeengine_b200 import _lib as L
    from tests.qconv import desc_for
    return desc_for(L, n, cin, h, w, cout, 1, 1, (1, 1), (0, 0, 0, 0))


@pytest.mark.parametrize("n, h, w, heads, d, documents", [
    (2, 9, 11, 4, 64, False), (1, 16, 16, 2, 72, False), (1, 20, 13, 4, 32, True)])
def test_block(n, h, w, heads, d, documents):
    import torch
    from computeengine_b200 import _lib as L
    g = torch.Generator(device="cuda").manual_seed(1)
    c, tokens = heads * d, n * h * w
    x = torch.randn(n, h, w, c, generator=g, device="cuda")
    gamma = 1 + 0.2 * torch.randn(c, generator=g, device="cuda")
    beta = 0.2 * torch.randn(c, generator=g, device="cuda")
    w_qkv = torch.randn(3 * c, c, generator=g, device="cuda") * c ** -0.5
    w_out = torch.randn(c, c, generator=g, device="cuda") * c ** -0.5
    b_qkv = 0.1 * torch.randn(3 * c, generator=g, device="cuda")
    dq, do = conv_desc(n, h, w, c, 3 * c), conv_desc(n, h, w, c, c)
    packed = []
    for dsc, wt in ((dq, w_qkv), (do, w_out)):
        p = torch.empty(int(L.lib.ie_cuda_f32_packed_weight_bytes(dsc)), dtype=torch.uint8,
                        device="cuda")
        L.check(L.lib.ie_cuda_f32_pack_weights(dsc, wt.data_ptr(), p.data_ptr(), stream()))
        packed.append(p)
    at = torch.arange(tokens, device="cuda") % (h * w)
    pos = torch.stack([at // w, at % w]).to(torch.int32)
    off = torch.tensor([0, 3 * w, tokens], dtype=torch.int32, device="cuda") if documents else None
    pairs = d // 4
    # the block
    split = torch.empty(n, h, w, 2 * c, dtype=torch.bfloat16, device="cuda")
    run_group_norm(L, group_norm_desc(L, x.shape, c, 8, 1e-5, L.IE_ACT_SILU, L.IE_DT_F32,
                                      L.IE_DT_BF16X2), x, gamma, beta, split)
    qkv = torch.empty(tokens, 3 * heads, d, device="cuda")
    L.check(L.lib.ie_cuda_conv2d_bf16x3(dq, L.IE_ACT_NONE, split.data_ptr(), packed[0].data_ptr(),
                                        b_qkv.data_ptr(), qkv.data_ptr(), L.IE_Y_F32_NHWC,
                                        stream()))
    rot = torch.empty(tokens, 3 * heads, d, dtype=torch.bfloat16, device="cuda")
    run_rotary(L, rotary_desc(L, qkv, rot, 2 * heads, (pairs, pairs), L.IE_ROTARY_AXIS_HALVES,
                              L.IE_ROTARY_FREQ_PER_AXIS, pos), qkv, pos, rot)
    b = 1 if documents else n
    q, k, v = (rot[:, i * heads:(i + 1) * heads].view(b, tokens // b, heads, d) for i in range(3))
    o = torch.empty(tokens, 2 * c, dtype=torch.bfloat16, device="cuda")
    ov = o.as_strided((b, tokens // b, heads, d), (tokens // b * 2 * c, 2 * c, d, 1))
    run_attention(L, attention_desc(L, q, k, v, ov, d ** -0.5, o_type=L.IE_DT_BF16X2),
                  attention_mask(L, 0, 2 if documents else 0, q_offsets=off, kv_offsets=off),
                  q, k, v, ov)
    y = torch.empty(n, h, w, c, device="cuda")
    L.check(L.lib.ie_cuda_conv2d_bf16x3_residual(do, L.IE_ACT_NONE, o.data_ptr(),
                                                 packed[1].data_ptr(), None, x.data_ptr(),
                                                 y.data_ptr(), L.IE_Y_F32_NHWC, stream()))
    assert L.take_device_error() == 0
    # the same in 64 bits, step by step on each step's own input
    gn, _ = group_norm_64(x.double(), 8, gamma, beta, 1e-5, 3)
    assert float((joined(split, c, c) - gn).abs().max()) <= 2.0 ** -14 * float(gn.abs().max())
    want = gn.reshape(tokens, c) @ w_qkv.double().t() + b_qkv.double()
    # the convolutions' own bar: 1e-3 of the largest value
    assert float((qkv.view(tokens, -1) - want).abs().max()) <= 1e-3 * float(want.abs().max())
    r64, size = rotary_64(qkv, pos, 2 * heads, (pairs, pairs), 2, 1)
    assert not ((rot.double() - r64).abs() > 2.0 ** -8 * r64.abs() + 2.0 ** -20 * size).any()
    a64, _, asize, _ = attention_64(q, k, v, d ** -0.5, q_offsets=off, kv_offsets=off)
    err = (joined(o, c, c).view(a64.shape) - a64).abs()
    assert not (err > 2.0 ** -8 * asize + 2.0 ** -12 * asize + 2.0 ** -16 * a64.abs()).any()
    y64 = joined(o, c, c) @ w_out.double().t() + x.double().view(tokens, c)
    assert float((y.view(tokens, c) - y64).abs().max()) <= 1e-3 * float(y64.abs().max())
