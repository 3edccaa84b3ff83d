"""Attention where one key outweighs each of many others by far and they still count
together: their weights, next to 1, are below what fp16 holds with all its bits (2^-14)
or at all (2^-25)."""
import math

import pytest

from tests.token_ops import (attention_64, attention_desc, attention_mask, check_attention,
                             run_attention)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("sq, hq, document", [(1, 2, False), (1, 2, True), (40, 2, False),
                                              (300, 2, True)])
@pytest.mark.parametrize("bits", [12, 16, 22, 25.5, 28])
@pytest.mark.parametrize("first", [True, False])
def test_a_tail_of_small_weights(first, bits, sq, hq, document, dtype):
    """The heavy key comes first or last; its value is 0, so o is all tail.  With the
    kernel's weights as large as 2^7 a weight of 2^-28 next to 1 is 2^-21, and 2^-22
    at the lower end of its spread: subnormal with a step of 2^-24, off by 2^-3 of it
    at most, either way, 2^-3 / sqrt(2^17) for the sum of all."""
    import torch
    from computeengine_b200 import _lib as L
    dt, n, d = getattr(torch, dtype), (1 << 17) + 5, 16
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.zeros(1, sq, hq, d, device="cuda")
    k = torch.zeros(1, n, 1, d, device="cuda")
    v = torch.rand(1, n, 1, d, generator=g, device="cuda") + 0.5
    at = 0 if first else n - 1
    q[..., 0], k[:, at, :, 0], v[:, at] = bits / 2, 2.0, 0.0
    # the others' scores spread over a factor of 4 around their place
    k[:, :, :, 1] = torch.rand(1, n, 1, generator=g, device="cuda") * 2 - 1
    k[:, at, :, 1] = 0
    q[..., 1] = 1.0
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    o, lse = torch.full_like(q, float("nan")), torch.full((1, hq, sq), float("nan"), device="cuda")
    kw = {}
    if document:
        off = lambda m: torch.tensor([0, m], dtype=torch.int32, device="cuda")  # noqa: E731
        kw = dict(q_offsets=off(sq), kv_offsets=off(n))
    m = attention_mask(L, documents=int(document), **kw)
    run_attention(L, attention_desc(L, q, k, v, o, math.log(2)), m, q, k, v, o, lse)
    assert not o.isnan().any()
    check_attention(o, lse, attention_64(q, k, v, math.log(2), **kw), dt)
