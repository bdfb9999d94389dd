"""The 4-bit KV cache operators at the edges of what they accept: scratch on
every boundary that is allowed, queries that are not finite or near the ends of
their range, probabilities far below the largest, sizes that take the rarer
paths.  References as in kv4_case.py."""

import numpy as np
import pytest
import torch

from kv4_case import DIM, Cache, i32

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def clear_status(cuda):
    import dial_b200

    dial_b200.device_status(clear=True)


def host(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


# ------------------------------------------------------------------- scratch
@pytest.mark.parametrize("queries", [1, 5, 200])
@pytest.mark.parametrize("weights", [False, True])
def test_scratch_on_every_sixteen_byte_boundary(cuda, queries, weights):
    """Scratch of exactly the stated size at each allowed start: the bits of a call
    that allocates its own, and nothing written beside it.  200 queries on 2600 slots
    are cut over the GPU, so that parts pass through the scratch."""
    from dial_b200 import kv4

    c = Cache(61, 2, 2600, 8, 2)
    base, table = c.device(cuda)
    q = (torch.randn(queries + 1, 8 * DIM, device=cuda) * 2).to(BF16)
    args = (table, i32(cuda, 1, 0), i32(cuda, 2600, 70), 2600, i32(cuda, 0, queries, queries + 1), queries)

    def call(scratch):
        cache = kv4.Kv4Cache(base.pages, base.weights.clone())
        out = kv4.kv4_attention(c.sh, cache, q, *args, accumulate=weights, scratch=scratch)
        return out, cache.weights

    want = call(None)
    o, b, _, _ = c.attend(host(q[:queries]), 1, 2600)
    assert (np.abs(host(want[0][:queries]) - o) <= b).all()
    n = kv4.attention_scratch_bytes(c.sh, 2, queries + 1, queries, 2600, weights)
    for start in (16, 32, 48, 64, 112, 128, 240):
        buf = torch.full((start + n + 256,), 0xA5, dtype=torch.uint8, device=cuda)
        assert buf.data_ptr() % 256 == 0
        got = call(buf[start:start + n])
        assert all(torch.equal(x, y) for x, y in zip(got, want)), start
        assert (buf[:start] == 0xA5).all() and (buf[start + n:] == 0xA5).all(), start
