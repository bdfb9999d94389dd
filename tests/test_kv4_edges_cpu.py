"""The 4-bit KV cache operators' host side at the edges of what they accept."""

import ctypes as C

import torch

from dial_b200 import _abi, kv4
from test_kv4_cpu import ATTN, EVICT, refused, shape


def test_single_queries_take_no_max_q():
    """Without q_starts every sequence has one query, whatever max_q says: such a call
    is not taken for one that has nothing to do."""
    args = {**ATTN, "sh": shape(), "starts": None, "rows": 2, "max_q": 0, "scratch": None}
    rc, msg = refused("dial_b200_kv4_attention", *args.values())
    assert rc == _abi.DIAL_ERR_INVALID and "scratch must be" in msg, (rc, msg)


def test_scratch_sizes_of_calls_that_are_refused():
    """The size functions refuse what the calls refuse: rows times heads, and entries
    to keep, beyond 31 bits."""
    sh = kv4.make_shape(64, 8, 64, 64)
    size = _abi.lib.dial_b200_kv4_attention_scratch_bytes
    most = 2 ** 31 // 64
    rc, _ = refused("dial_b200_kv4_attention", *{**ATTN, "sh": shape(q_heads=64), "rows": most, "q_ld": 8192,
                                                 "out_ld": 8192}.values())
    assert rc == _abi.DIAL_ERR_INVALID
    assert size(C.byref(sh), 2, most, 5, 64, 1) == -1 and size(C.byref(sh), 2, most - 1, 5, 64, 1) > 0
    size = _abi.lib.dial_b200_kv4_evict_scratch_bytes
    rc, _ = refused("dial_b200_kv4_evict", *{**EVICT, "sh": shape(), "keep": 2 ** 31}.values())
    assert rc == _abi.DIAL_ERR_INVALID
    assert size(C.byref(sh), 2, 64, 2 ** 31) == -1 and size(C.byref(sh), 2, 64, 2 ** 31 - 1) > 0


def test_one_row_of_any_stride():
    """A single row has no stride to be refused for."""
    x = torch.zeros(3, 515, dtype=torch.bfloat16)
    for row in (x[:1, :512], x[:0, :512], x.t()[:512].t()[:1], torch.zeros(512, 1, dtype=torch.bfloat16).t()):
        assert row.shape[1] == 512
        assert kv4._rows("q", row, torch.bfloat16, None, 512, -1) == (row.data_ptr(), 512)
    assert kv4._rows("q", x[:2, :512], torch.bfloat16, 2, 512, -1) == (x.data_ptr(), 515)
