"""A single block over so many keys that it runs for longer than the limit of one
of its waits (1 s)."""
import math

import pytest

from tests.token_ops import attention_desc, attention_mask, run_attention

pytestmark = pytest.mark.gpu


def test_a_block_that_runs_for_seconds():
    """One document of 2^28 - 37 keys, 4 GB of them: a document's keys are not
    shared out.  All keys are zero, so each weight is 1 and the sum counts the keys."""
    import torch
    from computeengine_b200 import _lib as L
    n = (1 << 28) - 37
    q = torch.ones(1, 1, 1, 8, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(1, n, 1, 8, dtype=torch.bfloat16, device="cuda")
    v = torch.ones_like(k)
    o, lse = torch.zeros_like(q), torch.zeros(1, 1, 1, device="cuda")
    at = lambda x: torch.tensor([0, x], dtype=torch.int32, device="cuda")  # noqa: E731
    q_off, kv_off = at(1), at(n)
    m = attention_mask(L, documents=1, q_offsets=q_off, kv_offsets=kv_off)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    run_attention(L, attention_desc(L, q, k, v, o, 1.0), m, q, k, v, o, lse)
    end.record()
    torch.cuda.synchronize()
    assert L.take_device_error() == 0
    assert begin.elapsed_time(end) > 1000  # else this shows nothing
    assert (o != 0).all()  # written
    assert abs(lse.item() - math.log(n)) <= 2.0 ** -12
