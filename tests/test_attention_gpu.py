"""ie_cuda_attention against the definition in 64 bits (tolerances: see
token_ops.check_attention)."""
import math

import pytest

from tests.token_ops import (HALF_STEP, attention_64, attention_desc, attention_mask,
                             check_attention, ptr, run_attention, stream)

pytestmark = pytest.mark.gpu

DTYPES = ["bfloat16", "float16"]


def tensors(b, sq, sk, hq, hk, d, dtype="bfloat16", seed=0, gain=2.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    q = (gain * torch.randn(b, sq, hq, d, generator=g, device="cuda")).to(dt)
    k = torch.randn(b, sk, hk, d, generator=g, device="cuda").to(dt)
    v = torch.randn(b, sk, hk, d, generator=g, device="cuda").to(dt)
    return q, k, v


def ints(*values):
    import torch
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def slopes_for(h):
    import torch
    return 2.0 ** -(8.0 * torch.arange(1, h + 1, device="cuda", dtype=torch.float32) / h)


def run_and_check(q, k, v, softcap=0.0, causal=0, kv_lens=None, prefix=None, q_offsets=None,
                  kv_offsets=None, slopes=None, with_lse=True, scale=None):
    import torch
    from computeengine_b200 import _lib as L
    scale = q.shape[3] ** -0.5 if scale is None else scale
    o = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), 7.0, device="cuda") if with_lse else None
    d = attention_desc(L, q, k, v, o, scale, softcap)
    docs = 0 if q_offsets is None else q_offsets.numel() - 1
    m = attention_mask(L, causal, docs, kv_lens, prefix, q_offsets, kv_offsets, slopes)
    run_attention(L, d, m, q, k, v, o, lse)
    assert L.take_device_error() == 0
    lens = None if kv_lens is None else kv_lens.clamp(0, k.shape[1])
    want = attention_64(q, k, v, scale, softcap, causal, lens, prefix, q_offsets, kv_offsets,
                        slopes)
    check_attention(o, lse, want, q.dtype)
    rows = want[3]
    assert (o[~rows] == 7).all()
    if with_lse:
        assert (lse.transpose(1, 2)[~rows] == 7).all()
    return o, lse, want


# lengths around every tile edge, one token, more queries than keys, long keys
LENGTHS = [(1, 1), (1, 2), (1, 16), (1, 17), (1, 127), (1, 129), (1, 1000), (2, 2), (7, 64),
           (16, 16), (17, 80), (33, 33), (64, 65), (77, 77), (127, 128), (128, 127), (129, 300),
           (200, 77), (255, 256), (257, 257), (384, 640), (513, 511), (1000, 1)]


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("sq, sk", LENGTHS, ids=str)
def test_lengths(sq, sk, causal):
    """More queries than keys and causal: the first rows see nothing."""
    run_and_check(*tensors(2, sq, sk, 4, 2, 64, seed=sq + sk), causal=causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 5, 8, 16, 24, 31, 32, 40, 63, 64, 72, 80, 96, 100, 112, 120, 127,
                               128])
@pytest.mark.parametrize("sq, sk", [(1, 150), (10, 150), (150, 150)], ids=str)
def test_head_dims(sq, sk, d, dtype):
    run_and_check(*tensors(1, sq, sk, 3, 1, d, dtype, seed=d), causal=1)


@pytest.mark.parametrize("sq, sk", [(1, 700), (5, 300), (140, 300)], ids=str)
@pytest.mark.parametrize("hq, hk", [(1, 1), (3, 3), (8, 1), (12, 4), (71, 1), (40, 8), (6, 2),
                                    (16, 1), (17, 1), (32, 1)], ids=str)
def test_heads(hq, hk, sq, sk):
    run_and_check(*tensors(2, sq, sk, hq, hk, 64, seed=hq), causal=1, slopes=slopes_for(hq))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("options", ["cap", "bias", "cap bias", "cap causal", "bias causal",
                                     "cap bias causal prefix", "prefix causal"])
@pytest.mark.parametrize("sq, sk, d", [(1, 333, 128), (9, 333, 80), (333, 333, 128), (260, 390, 64)],
                         ids=str)
def test_scores_and_masks(sq, sk, d, options, dtype):
    q, k, v = tensors(3, sq, sk, 4, 2, d, dtype, seed=3, gain=4.0)
    run_and_check(q, k, v, softcap=15.0 if "cap" in options else 0.0, causal=int("causal" in options),
                  slopes=slopes_for(4) if "bias" in options else None,
                  prefix=ints(0, 200, 1000) if "prefix" in options else None)


@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0, 1000.0])
def test_cap_over_its_range(cap):
    """Scores far below, around and far above the cap."""
    for gain in (0.5, 8.0, 100.0):
        for sq in (1, 130):
            q, k, v = tensors(1, sq, 300, 2, 2, 64, seed=4, gain=gain)
            if cap == 1000.0 and gain == 100.0:
                continue  # scores of hundreds: one step of a score is over the tolerance
            run_and_check(q, k, v, softcap=cap)


@pytest.mark.parametrize("sq", [1, 3, 20, 150])
def test_ragged_lengths_with_garbage_behind_them(sq):
    """NaN and infinities behind each sequence's length reach nothing; empty
    sequences give zeros; lengths out of range are clamped."""
    import torch
    q, k, v = tensors(7, sq, 400, 8, 2, 128, seed=5)
    lens = ints(400, 1, 0, 129, 255, 128, 999)
    for n, l in enumerate(lens.tolist()):
        k[n, l:] = float("nan")
        v[n, l:] = float("inf") if n % 2 else float("nan")
    for causal in (0, 1):
        o, lse, _ = run_and_check(q, k, v, causal=causal, kv_lens=lens, softcap=30.0)
        assert not o[2].any() and torch.isinf(lse[2]).all()


@pytest.mark.parametrize("sq", [1, 130])
def test_negative_length_is_empty(sq):
    q, k, v = tensors(2, sq, 64, 2, 2, 64)
    run_and_check(q, k, v, kv_lens=ints(-5, 64))


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("cuts", [
    (0, 500), (0, 1, 2, 3, 500), (0, 0, 130, 130, 257, 480), (10, 20, 300), (0, 128, 256, 384, 500),
    (0, 127, 255, 500), (0, 0, 0), (500, 500), tuple(range(0, 501, 10)),
], ids=str)
def test_documents(cuts, causal):
    """Documents that end inside tiles, of length 0 and 1; rows before the first
    and behind the last left as they were."""
    off = ints(*cuts)
    q, k, v = tensors(1, 500, 500, 4, 4, 72, seed=6)
    run_and_check(q, k, v, causal=causal, q_offsets=off, kv_offsets=off)
    run_and_check(q, k, v, causal=causal, q_offsets=off, kv_offsets=off, slopes=slopes_for(4),
                  prefix=ints(*[7 * i % 50 for i in range(len(cuts) - 1)]) if causal else None)


def test_documents_do_not_leak():
    """A document of NaN harms no other."""
    import torch
    off = ints(0, 100, 230, 400)
    q, k, v = tensors(1, 400, 400, 2, 2, 64, seed=7)
    for t in (k, v):
        t[0, 100:230] = float("nan")
    o = torch.empty_like(q)
    from computeengine_b200 import _lib as L
    d = attention_desc(L, q, k, v, o, 0.125)
    run_attention(L, d, attention_mask(L, 0, 3, q_offsets=off, kv_offsets=off), q, k, v, o)
    assert torch.isnan(o[0, 100:230]).all()
    assert not torch.isnan(o[0, :100]).any() and not torch.isnan(o[0, 230:]).any()


def test_documents_of_different_lengths():
    """Queries of each document are the last of its keys (cached keys before)."""
    q_off, kv_off = ints(0, 1, 5, 5, 140), ints(0, 300, 310, 350, 700)
    q, k, v = tensors(1, 150, 720, 8, 2, 64, seed=8)
    for causal in (0, 1):
        run_and_check(q, k, v, causal=causal, q_offsets=q_off, kv_offsets=kv_off, softcap=20.0)


def test_many_documents():
    import torch
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 9, (700,), generator=g)
    off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32).cuda()
    n = int(off[-1]) + 3
    run_and_check(*tensors(1, n, n, 2, 1, 64, seed=9), causal=1, q_offsets=off, kv_offsets=off)


@pytest.mark.parametrize("sq", [1, 140])
def test_extreme_scores(sq):
    """Rows whose scores are all far below, far above, and equal; a slope that
    leaves one key; a row whose only visible scores are -inf."""
    import torch
    q, k, v = tensors(1, sq, 300, 2, 2, 64, seed=10)
    run_and_check(q, k, v, scale=0.0)
    run_and_check(q, k, v, slopes=torch.full((2,), 1000.0, device="cuda"))
    k[0, :, 0] = -60000.0 if q.dtype == torch.float16 else -1e30
    q[0, :, 0] = 1.0
    run_and_check(q, k * 0 + k[:, :, :, :1] * 0 - 100.0, v, scale=1.0)
    from computeengine_b200 import _lib as L
    k[..., 0] = float("-inf")
    q.fill_(1.0)
    o, lse = torch.full_like(q, 7.0), torch.zeros(1, 2, sq, device="cuda")
    run_attention(L, attention_desc(L, q, k, v, o, 1.0), None, q, k, v, o, lse)
    assert not o.any() and (lse == float("-inf")).all()


@pytest.mark.parametrize("sq", [1, 140])
def test_nan_in_a_visible_place_shows(sq):
    import torch
    from computeengine_b200 import _lib as L
    q, k, v = tensors(1, sq, 300, 2, 2, 64, seed=11)
    k[0, 77, 1, 3] = float("nan")
    o = torch.zeros_like(q)
    run_attention(L, attention_desc(L, q, k, v, o, 0.125), None, q, k, v, o)
    assert torch.isnan(o[:, :, 1]).all() and not torch.isnan(o[:, :, 0]).any()


ORDERS = ["heads first", "packed qkv", "padded rows", "unaligned", "broadcast heads", "odd stride"]


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("sq, sk", [(1, 200), (12, 200), (200, 200)], ids=str)
def test_strides(sq, sk, order):
    import torch
    from computeengine_b200 import _lib as L
    b, hq, hk, d = 2, 4, 2, 64
    q, k, v = tensors(b, sq, sk, hq, hk, d, seed=12)
    o = torch.full_like(q, 7.0)
    if order == "heads first":
        q, k, v, o = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, o))
    elif order == "packed qkv":
        kv = torch.cat([k, v], 2)
        k, v = kv[:, :, :hk], kv[:, :, hk:]
    elif order == "padded rows":
        q, k, v, o = (torch.nn.functional.pad(t, (0, 16))[..., :d] for t in (q, k, v, o))
    elif order == "unaligned":
        q, k, v, o = (torch.nn.functional.pad(t, (1, 7))[..., 1:d + 1] for t in (q, k, v, o))
    elif order == "broadcast heads":
        k, v = (t[:, :, :1].expand(b, sk, hk, d) for t in (k, v))
    else:
        q, k, v, o = (torch.nn.functional.pad(t, (0, 3))[..., :d] for t in (q, k, v, o))
    base = o._base if o._base is not None else o
    base.fill_(7.0)
    dsc = attention_desc(L, q, k, v, o, 0.125)
    lse = torch.zeros(b, hq, sq, device="cuda")
    run_attention(L, dsc, attention_mask(L, 1), q, k, v, o, lse)
    check_attention(o, lse, attention_64(q, k, v, 0.125, causal=1), q.dtype)
    if order in ("padded rows", "unaligned", "odd stride"):
        mark = torch.full_like(base, 1.0)
        mark.as_strided(o.shape, o.stride(), o.storage_offset()).zero_()
        assert (base[mark.bool()] == 7).all()


@pytest.mark.parametrize("sq", [1, 13, 200])
@pytest.mark.parametrize("d", [64, 72])
def test_split_output(sq, d):
    """BF16X2 output: hi + lo, what ie_cuda_conv2d_bf16x3 reads."""
    import torch
    from computeengine_b200 import _lib as L
    hq, plane = 4, (4 * d + 15) // 16 * 16
    q, k, v = tensors(2, sq, 200, hq, 2, d, seed=13)
    o = torch.full((2, sq, 2 * plane), 7.0, dtype=torch.bfloat16, device="cuda")
    view = o.as_strided((2, sq, hq, d), (sq * 2 * plane, 2 * plane, d, 1))
    dsc = attention_desc(L, q, k, v, view, d ** -0.5, o_type=L.IE_DT_BF16X2)
    run_attention(L, dsc, None, q, k, v, view)
    want, _, size, _ = attention_64(q, k, v, d ** -0.5)
    got = (o[..., :hq * d].double() + o[..., plane:plane + hq * d].double()).view(2, sq, hq, d)
    # the weights are bf16 all the same; the output's own rounding is 2^-16
    tol = HALF_STEP[torch.bfloat16] * size + 2.0 ** -16 * want.abs() + 2.0 ** -12 * size
    assert not ((got - want).abs() > tol).any()
    assert (o[..., hq * d:plane] == 7).all() and (o[..., plane + hq * d:] == 7).all()


@pytest.mark.parametrize("sq, sk, b, hk", [(1, 40000, 1, 1), (1, 9001, 3, 2), (4, 20000, 1, 2),
                                           (150, 12000, 1, 1), (1, 4096, 32, 8)], ids=str)
def test_long_axis(sq, sk, b, hk):
    run_and_check(*tensors(b, sq, sk, 4 * hk, hk, 128, seed=14), causal=1, softcap=50.0)


@pytest.mark.parametrize("sq, sk", [(1, 5000), (9, 3000), (300, 300)], ids=str)
def test_repeatable(sq, sk):
    import torch
    q, k, v = tensors(2, sq, sk, 8, 2, 128, seed=15)
    a = run_and_check(q, k, v, causal=1)
    b = run_and_check(q, k, v, causal=1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_cache_past_32_bits():
    """The keys of the last sequence lie past 2^32 bytes; alone it gives the same."""
    import torch
    from computeengine_b200 import _lib as L
    b, sk, hk, d = 5, 70000, 32, 128
    k = torch.zeros(b, sk, hk, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    q1, k1, v1 = tensors(1, 1, sk, hk, hk, d, seed=16)
    k[-1], v[-1] = k1[0], v1[0]
    for sq in (1, 40):
        q = torch.randn(b, sq, hk, d, device="cuda").bfloat16()
        o, one = torch.empty_like(q), torch.empty_like(q[-1:])
        run_attention(L, attention_desc(L, q, k, v, o, 0.1), attention_mask(L, 1), q, k, v, o)
        ql = q[-1:].contiguous()
        want = attention_64(ql, k1, v1, 0.1, causal=1)
        check_attention(o[-1:], None, want, q.dtype)
        assert not o[:-1].any()


@pytest.mark.parametrize("sq, sk", [(1, 5000), (200, 200)], ids=str)
def test_captured_replayed_and_concurrent(sq, sk):
    """Two graphs with a workspace each, replayed on two streams at once, over
    inputs and lengths that change between replays."""
    import torch
    from computeengine_b200 import _lib as L
    runs = []
    for n in range(2):
        q, k, v = tensors(2, sq, sk, 8, 2, 128, seed=17 + n)
        lens = ints(sk, sk // 2)
        o, lse = torch.empty_like(q), torch.empty(2, 8, sq, device="cuda")
        d = attention_desc(L, q, k, v, o, 0.125)
        m = attention_mask(L, 1, kv_lens=lens)
        ws = torch.empty(max(int(L.lib.ie_cuda_attention_workspace_bytes(d, m)), 1),
                         dtype=torch.uint8, device="cuda")
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            L.check(L.lib.ie_cuda_attention(d, m, *(t.data_ptr() for t in (q, k, v, o, lse, ws)),
                                            ws.numel(), stream()))
        runs.append((q, k, v, lens, o, lse, ws, s, g))
    for step in range(3):
        for q, _, _, lens, *_ in runs:
            q.mul_(1.1)
            lens.sub_(step)
        torch.cuda.synchronize()
        for *_, s, g in runs:
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for q, k, v, lens, o, lse, *_ in runs:
            check_attention(o, lse, attention_64(q, k, v, 0.125, causal=1, kv_lens=lens), q.dtype)


def test_workspace_refusals():
    import torch
    from computeengine_b200 import _lib as L
    q, k, v = tensors(1, 1, 8192, 8, 2, 128)
    o = torch.empty_like(q)
    d = attention_desc(L, q, k, v, o, 0.1)
    need = int(L.lib.ie_cuda_attention_workspace_bytes(d, None))
    if need == 0:
        pytest.skip("one sequence of this length is not split")
    ws = torch.empty(need + 256, dtype=torch.uint8, device="cuda")
    f, args = L.lib.ie_cuda_attention, [t.data_ptr() for t in (q, k, v, o)]
    assert f(d, None, *args, None, None, need, stream()) == L.IE_INVALID_ARGUMENT
    assert f(d, None, *args, None, ws.data_ptr(), need - 1, stream()) == L.IE_INVALID_ARGUMENT
    assert f(d, None, *args, None, ws.data_ptr() + 8, need, stream()) == L.IE_INVALID_ARGUMENT
    assert f(d, None, *args, None, ws.data_ptr(), need, stream()) == L.IE_OK
    torch.cuda.synchronize()


def test_operator():
    import torch
    from computeengine_b200.ops import AttentionOp, Code
    q, k, v = tensors(2, 50, 60, 4, 2, 64, "float16", seed=18)
    lens, sl = ints(60, 31), slopes_for(4)
    op = AttentionOp()
    assert op.configure({"causal": True, "softcap": 25.0})
    out = [None, None]
    st = op.forward([q, k, v, lens, None, None, None, sl], out)
    assert st, st.message
    check_attention(out[0], out[1],
                    attention_64(q, k, v, 0.125, 25.0, 1, lens, slopes=sl), q.dtype)
    off = ints(0, 20, 45)
    out = [None]
    assert op.forward([q[:1], k[:1, :50], v[:1, :50], None, None, off, off], out)
    check_attention(out[0], None, attention_64(q[:1], k[:1, :50], v[:1, :50], 0.125, 25.0, 1,
                                               q_offsets=off, kv_offsets=off), q.dtype)
    assert not out[0][0, 45:].any()
    for bad, code in (([q, k], Code.InvalidArgument), ([q, k, v[:, :5]], Code.InvalidArgument),
                      ([q.float(), k, v], Code.Unsupported),
                      ([q, k, v, lens.long()], Code.InvalidArgument),
                      ([q, k, v, lens[:1]], Code.InvalidArgument),
                      ([q, k, v, None, None, off, off], Code.InvalidArgument),
                      ([q, k, v, None, None, off, None], Code.InvalidArgument),
                      ([q, k[..., :32], v[..., :32]], Code.InvalidArgument),
                      ([q, k, v, lens.cpu()], Code.InvalidArgument),
                      ([q, k, v, None, None, None, None, sl[:2]], Code.InvalidArgument)):
        o = [None]
        st = op.forward(bad, o)
        assert not st and st.code == code and o == [None], bad


@pytest.mark.parametrize("q_len", [1, 17])
def test_bias_of_near_keys_behind_2_24(q_len):
    """The distance bias of keys next to their query, at places that fp32 does
    not hold: the last 2048 keys stand for all of them, as a key further away has
    at most e^(60 - 2047) of the weight of the nearest, which is zero.

    Tolerance of lse: distances below 2048 are exact and the products and
    exponentials of single scores are off by steps of scores below 2^7 for what
    weighs anything, 2^-16; scores of the running maximum alike."""
    import torch
    from computeengine_b200 import _lib as L
    n, d, tail = (1 << 24) + 1029, 8, 2048
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(1, n, 1, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(1, q_len, 1, d, generator=g, device="cuda").bfloat16()
    slopes = torch.tensor([1.0], device="cuda")
    o = torch.empty_like(q)
    lse = torch.empty(1, 1, q_len, device="cuda")
    desc = attention_desc(L, q, k, k, o, d ** -0.5)
    run_attention(L, desc, attention_mask(L, slopes=slopes), q, k, k, o, lse)
    near = k[:, n - tail:].double()[0, :, 0]
    s = desc.scale * q.double()[0, :, 0] @ near.T
    p = torch.arange(q_len, device="cuda") + tail - q_len
    s = s - (p[:, None] - torch.arange(tail, device="cuda")[None]).abs().double()
    want = torch.softmax(s, 1) @ near
    assert (lse[0, 0].double() - torch.logsumexp(s, 1)).abs().max() < 2.0 ** -14
    size = torch.softmax(s, 1) @ near.abs()
    tol = HALF_STEP[torch.bfloat16] * (want.abs() + size) + 2.0 ** -12 * size
    assert ((o[0, :, 0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("q_len", [1, 40])
def test_offsets_past_32_bits(q_len):
    """A batch row, and a token, more than 2^32 bytes and 2^31 elements away."""
    import torch
    from computeengine_b200 import _lib as L
    d, n, far = 64, 300, (1 << 31) + 4096
    store = torch.empty(far + 2 * n * d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(7)
    near = torch.randn(2, n, 1, d, generator=g, device="cuda").bfloat16()
    k = store.as_strided((2, n, 1, d), (far, d, d, 1))
    k.copy_(near)
    q = torch.randn(2, q_len, 1, d, generator=g, device="cuda").bfloat16()
    out = []
    for kk in (k, near):
        o = torch.empty_like(q)
        m = attention_mask(L, causal=1)
        run_attention(L, attention_desc(L, q, kk, kk, o, 0.125), m, q, kk, kk, o)
        out.append(o)
    assert torch.equal(*out)
    stride = (1 << 23) + 64
    k = store.as_strided((1, 257, 1, d), (stride, stride, d, 1))
    k.copy_(near[:1, :257])
    q, out = q[:1], []
    for kk in (k, near[:1, :257]):
        o = torch.empty_like(q)
        run_attention(L, attention_desc(L, q, kk, kk, o, 0.125), None, q, kk, kk, o)
        out.append(o)
    assert torch.equal(*out)
