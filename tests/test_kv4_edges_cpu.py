"""The 4-bit KV cache operators' host side at the edges of what they accept."""

from dial_b200 import _abi
from test_kv4_cpu import ATTN, refused, shape


def test_single_queries_take_no_max_q():
    """Without q_starts every sequence has one query, whatever max_q says: such a call
    is not taken for one that has nothing to do."""
    args = {**ATTN, "sh": shape(), "starts": None, "rows": 2, "max_q": 0, "scratch": None}
    rc, msg = refused("dial_b200_kv4_attention", *args.values())
    assert rc == _abi.DIAL_ERR_INVALID and "scratch must be" in msg, (rc, msg)
