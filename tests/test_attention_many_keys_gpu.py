"""Attention over so many keys of nearly equal weight that a sum of them is large
next to each.

The weights are equal and exact (q is 0), v is not negative: o is the mean of v,
off by one rounding to its type and by what the sums lose.  A tensor core cuts
off what lies below its fp32 sum's last place: of n products of about 1 at most
n * 2^-24 of each, so 2^-9 for the 2^15 keys that go through one such sum, and
half of that on average.  Everything else is rounded to nearest."""
import pytest

from tests.token_ops import HALF_STEP, attention_desc, attention_mask, run_attention

pytestmark = pytest.mark.gpu


def run(q, k, v, document):
    import math
    import torch
    from computeengine_b200 import _lib as L
    o = torch.full_like(q, float("nan"))
    lse = torch.full((q.shape[0], q.shape[2], q.shape[1]), float("nan"), device="cuda")
    m = attention_mask(L)
    if document:  # the keys of a document are not shared out
        at = [torch.tensor([0, n], dtype=torch.int32, device="cuda")
              for n in (q.shape[1], k.shape[1])]
        m = attention_mask(L, documents=1, q_offsets=at[0], kv_offsets=at[1])
    run_attention(L, attention_desc(L, q, k, v, o, 1.0), m, q, k, v, o, lse)
    assert L.take_device_error() == 0
    want = v.double().mean(dim=1, keepdim=True).repeat_interleave(q.shape[2] // v.shape[2], 2)
    err = ((o.double() - want).abs() / want).max()
    assert err <= HALF_STEP[q.dtype] + 2.0 ** -10, float(err)
    assert (lse - math.log(k.shape[1])).abs().max() <= 2.0 ** -12


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("keys", [(1 << 15) + 1, 1 << 18, (1 << 20) + 77, 1 << 23])
@pytest.mark.parametrize("sq, hq, hk, document", [(1, 1, 1, False), (1, 1, 1, True),
                                                  (3, 8, 2, False), (40, 4, 2, False),
                                                  (300, 2, 1, True)])
def test_equal_weights(sq, hq, hk, document, keys, dtype):
    """Single tokens with and without shares, packed rows with shares, whole tiles."""
    import torch
    dt = getattr(torch, dtype)
    for d in (8, 72) if keys < 1 << 20 else (8,):
        g = torch.Generator(device="cuda").manual_seed(keys)
        v = (torch.rand(1, keys, hk, d, generator=g, device="cuda") + 0.5).to(dt)
        run(torch.zeros(1, sq, hq, d, dtype=dt, device="cuda"), torch.zeros_like(v), v, document)


@pytest.mark.parametrize("document", [False, True])
def test_equal_weights_of_rows_that_tma_cannot_read(document):
    import torch
    v = torch.rand(1, 1 << 20, 1, 9, device="cuda")[..., 1:].add(0.5).to(torch.float16)
    v = torch.cat([v[..., :1], v], -1)[..., 1:]  # rows of 18 bytes
    q = torch.zeros(1, 5, 1, 8, dtype=torch.float16, device="cuda")
    run(q, torch.zeros_like(v), v, document)


@pytest.mark.parametrize("sq, document", [(1, False), (40, False), (300, True)])
def test_growing_scores_over_many_keys(sq, document):
    """The maximum moves all the time, between and at the points where the sums
    are put away; a causal border and a cap besides.  Against 64 bits."""
    import torch
    from computeengine_b200 import _lib as L
    from tests.token_ops import attention_64, check_attention
    n = 70001
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.rand(1, sq, 2, 64, generator=g, device="cuda").bfloat16()
    k = torch.rand(1, n, 1, 64, generator=g, device="cuda")
    k = (k * torch.linspace(0, 1, n, device="cuda")[None, :, None, None]).bfloat16()
    v = torch.randn(1, n, 1, 64, generator=g, device="cuda").bfloat16()
    o, lse = torch.empty_like(q), torch.empty(1, 2, sq, device="cuda")
    at = [torch.tensor([0, x], dtype=torch.int32, device="cuda") for x in (sq, n)]
    kw = dict(causal=1)
    if document:
        kw.update(q_offsets=at[0], kv_offsets=at[1])
    m = attention_mask(L, documents=int(document), **kw)
    for cap in (0.0, 30.0):
        run_attention(L, attention_desc(L, q, k, v, o, 2.0, cap), m, q, k, v, o, lse)
        assert not o.isnan().any()
        check_attention(o, lse, attention_64(q, k, v, 2.0, cap, **kw), q.dtype)


@pytest.mark.parametrize("options", ["plain", "bias", "cap", "prefix", "cap bias"])
@pytest.mark.parametrize("batch, sq, hq, hk, keys, dtype", [
    (1, 130, 80, 1, 70001, "bfloat16"),    # blocks enough without shares
    (3, 130, 30, 2, 66000, "float16"),     # the same over ragged lengths
    (1, 130, 70, 1, 140000, "bfloat16"),   # two shares, each put away twice
    (1, 40, 148, 2, 140000, "float16"),    # several heads in a tile
])
def test_long_keys_under_masks(batch, sq, hq, hk, keys, dtype, options):
    """The first and last heads against 64 bits; the score's maximum moves along the
    keys; a split output stands for the same values."""
    import torch
    from computeengine_b200 import _lib as L
    from tests.token_ops import attention_64, check_attention, joined
    g = torch.Generator(device="cuda").manual_seed(keys + sq)
    dt, d = getattr(torch, dtype), 64
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    q, v = (rand(batch, sq, hq, d) * 2).to(dt), rand(batch, keys, hk, d).to(dt)
    grow = torch.linspace(0.2, 1.5, keys, device="cuda")[None, :, None, None]
    k = (rand(batch, keys, hk, d) * grow).to(dt)
    slopes = 2.0 ** -(8.0 + 6.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kw = dict(causal=1)
    if batch == 3:
        kw.update(kv_lens=ints(keys, 40000, 100))
    if "prefix" in options:
        kw.update(prefix=ints(*[keys] * batch))
    if "bias" in options:
        kw.update(slopes=slopes)
    cap = 40.0 if "cap" in options else 0.0
    o, lse = torch.empty_like(q), torch.empty(batch, hq, sq, device="cuda")
    m = attention_mask(L, **kw)
    run_attention(L, attention_desc(L, q, k, v, o, d ** -0.5, cap), m, q, k, v, o, lse)
    assert L.take_device_error() == 0
    assert not o.isnan().any()
    for h, c in ((0, 0), (hq - 1, hk - 1)):
        part = dict(kw, slopes=slopes[h:h + 1]) if "bias" in options else kw
        want = attention_64(q[:, :, h:h + 1], k[:, :, c:c + 1], v[:, :, c:c + 1], d ** -0.5, cap,
                            **part)
        check_attention(o[:, :, h:h + 1], lse[:, h:h + 1], want, dt)
    if dt == torch.bfloat16:
        two = torch.empty(batch, sq, 2 * hq * d, dtype=dt, device="cuda")
        desc = attention_desc(L, q, k, v, o, d ** -0.5, cap, o_type=L.IE_DT_BF16X2)
        for i, s in enumerate((sq * 2 * hq * d, 2 * hq * d, d)):
            desc.o_stride[i] = s
        run_attention(L, desc, m, q, k, v, two, None)
        both = joined(two, hq * d, hq * d).reshape(o.shape)
        # one rounding to bf16 apart, and the lo plane's own
        assert ((both - o.double()).abs() <= (2.0 ** -8 + 2.0 ** -16) * both.abs() + 2.0 ** -126).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("weight", [0.3, 0.7071])
@pytest.mark.parametrize("sq, batch, document, keys", [
    (20, 1, True, 1 << 26), (300, 1, True, 1 << 24), (1, 1, False, 1 << 26),
    (1, 300, False, 1 << 20), (40, 80, False, 1 << 19)])
def test_equal_weights_that_round(sq, batch, document, keys, weight, dtype):
    """The first key's weight is 1 and its value 0, all others weigh the same and hold 1:
    each addition to a long sum rounds the same way.  The scores' spread is exact to
    2^-22, the weights' sum to 2^-12 (lse) and o to a few 2^-12 besides its rounding."""
    import math
    import torch
    from computeengine_b200 import _lib as L
    dt = getattr(torch, dtype)
    scale = -math.log(weight)
    v = torch.ones(batch, keys, 1, 8, dtype=dt, device="cuda")
    k = torch.zeros_like(v)
    k[:, 0, :, 0], v[:, 0] = 1, 0
    q = torch.zeros(batch, sq, 1, 8, dtype=dt, device="cuda")
    q[..., 0] = 1
    o = torch.zeros_like(q)
    lse = torch.zeros(batch, 1, sq, device="cuda")
    m = attention_mask(L)
    if document:
        at = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (sq, keys)]
        m = attention_mask(L, documents=1, q_offsets=at[0], kv_offsets=at[1])
    run_attention(L, attention_desc(L, q, k, v, o, scale), m, q, k, v, o, lse)
    assert L.take_device_error() == 0
    total = 1 + (keys - 1) * math.exp(-scale)
    assert (lse.double() - (math.log(total) + scale)).abs().max() <= 2.0 ** -12
    want = (total - 1) / total
    assert (o.double() - want).abs().max() <= HALF_STEP[dt] + 2.0 ** -11
