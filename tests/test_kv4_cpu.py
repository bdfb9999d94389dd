"""Refusals of the 4-bit KV cache operators, before any device work, and the
reference's own codec against the formats' definitions."""

import ctypes as C

import numpy as np
import pytest
import torch

import dial_b200
from dial_b200 import _abi, kv4
from kv4_case import E2M1, E4M3, Cache, decode, encode, nearest, pack, unpack

P = 1 << 20  # an aligned address that nothing reads


def refused(name, *args):
    buf = C.create_string_buffer(512)
    rc = getattr(_abi.lib, name)(*args, buf, 512)
    return rc, buf.value.decode()


def shape(**kw):
    sh = kv4.make_shape(32, 8, 64, 640, max_pos=4096)
    for k, v in kw.items():
        setattr(sh, k, v)
    return C.byref(sh)


APPEND = dict(sh=None, qkv=P, qkv_ld=48 * 128, qn=P, kn=P, cos=P, sin=P, pages=P, weights=P, pp=P, bt=P,
              sessions=4, sids=P, slots=P, pos=P, q_out=P, q_ld=32 * 128, rows=3, stream=None)
READ = dict(sh=None, pages=P, bt=P, sessions=4, sids=P, first=None, lens=P, seqs=2, count=5, k=P, v=P,
            stream=None)
ATTN = dict(sh=None, q=P, q_ld=4096, pages=P, weights=P, bt=P, sessions=4, sids=P, lens=P, starts=P,
            seqs=2, rows=9, max_q=5, max_len=1024, out=P, out_ld=4096, scratch=P, stream=None)
EVICT = dict(sh=None, pages=P, weights=P, pp=P, bt=P, dst=None, sessions=4, sids=P, lens=P, lens_out=P,
             seqs=2, max_len=1024, keep=512, recent=32, scratch=P, stream=None)
POOL = [({"sh": dict(head_dim=64)}, "head_dim must be 128"), ({"sh": dict(q_heads=30)}, "times kv_heads"),
        ({"sh": dict(q_heads=8 * 17)}, "times kv_heads"), ({"sh": dict(kv_heads=0)}, "times kv_heads"),
        ({"sh": dict(max_blocks=0)}, "out of range"), ({"sh": dict(num_blocks=0)}, "out of range"),
        ({"sh": dict(k_scale=0.0)}, "must be positive"),
        ({"sh": dict(v_scale=float("nan"))}, "must be positive"), ({"sh": dict(act=2)}, "act must be"),
        ({"sessions": 0}, "sessions 0"), ({"pages": P + 8}, "16-byte aligned"),
        ({"pages": None}, "null pointer"), ({"bt": None}, "null pointer"), ({"sids": None}, "null pointer")]
CASES = [("append", APPEND, c) for c in POOL + [
    ({"qkv": None}, "null pointer"), ({"slots": None}, "null pointer"), ({"qn": None}, "go in pairs"),
    ({"cos": None}, "go in pairs"), ({"pos": None}, "need positions"),
    ({"sh": dict(max_pos=0)}, "max_pos 0"), ({"sh": dict(eps=-1.0)}, "eps"), ({"rows": -1}, "rows -1"),
    ({"qkv_ld": 47 * 128}, "must hold their heads"), ({"qkv_ld": 48 * 128 + 4}, "16-byte"),
    ({"qkv": P + 8}, "16-byte"), ({"q_ld": 100}, "must hold"), ({"kn": P + 8}, "16-byte aligned")]]
CASES += [("read", READ, c) for c in POOL + [
    ({"lens": None}, "null pointer"), ({"k": None}, "null pointer"), ({"v": P + 8}, "16-byte"),
    ({"count": -1}, "out of range"), ({"seqs": -1}, "out of range"),
    ({"seqs": 1 << 20, "count": 1 << 20}, "out of range")]]
CASES += [("attention", ATTN, c) for c in POOL + [
    ({"q": None}, "null pointer"), ({"out": None}, "null pointer"), ({"lens": None}, "null pointer"),
    ({"seqs": 65536}, "seqs 65536"), ({"rows": -1}, "rows -1"), ({"starts": None}, "must equal seqs"),
    ({"max_len": 1025}, "exceeds the block table"), ({"max_q": -1}, "max_q -1"),
    ({"sh": dict(softmax_scale=-1.0)}, "softmax_scale"), ({"q_ld": 4095}, "must hold"),
    ({"out_ld": 4100}, "16-byte"), ({"q": P + 8}, "16-byte"), ({"scratch": None}, "scratch must be")]]
CASES += [("evict", EVICT, c) for c in POOL + [
    ({"weights": None}, "null pointer"), ({"lens_out": None}, "null pointer"),
    ({"seqs": -1}, "seqs -1"), ({"max_len": 2000}, "exceeds the block table"),
    ({"keep": -1}, "keep -1"), ({"recent": 513}, "recent <= keep"), ({"pp": None}, "needs positions"),
    ({"scratch": None}, "scratch must be")]]


@pytest.mark.parametrize("name,base,case", CASES, ids=lambda v: str(v)[:48] if not isinstance(v, dict) else "")
def test_bad_arguments_are_refused_before_device_work(name, base, case):
    change, text = case
    args = {**base, **change}
    args["sh"] = shape(**change.get("sh", {}))
    rc, msg = refused("dial_b200_kv4_" + name, *args.values())
    assert rc == _abi.DIAL_ERR_INVALID and text in msg, (rc, msg)


@pytest.mark.parametrize("name,base,none", [("append", APPEND, {"rows": 0}), ("read", READ, {"count": 0}),
                                            ("read", READ, {"seqs": 0}), ("attention", ATTN, {"seqs": 0}),
                                            ("attention", ATTN, {"rows": 0}), ("evict", EVICT, {"seqs": 0})])
def test_empty_calls_do_nothing(name, base, none):
    args = {**base, **none}
    args["sh"] = shape()
    assert refused("dial_b200_kv4_" + name, *args.values())[0] == _abi.DIAL_OK


def test_null_shape_and_sizes():
    assert refused("dial_b200_kv4_read", *{**READ, "sh": None}.values())[0] == _abi.DIAL_ERR_INVALID
    assert _abi.lib.dial_b200_kv4_attention_scratch_bytes(None, 1, 1, 1, 1, 0) == -1
    assert _abi.lib.dial_b200_kv4_evict_scratch_bytes(None, 1, 1, 1) == -1
    sh = kv4.make_shape(32, 8, 64, 640)
    assert kv4.attention_scratch_bytes(sh, 4, 4, 1, 1024, True) >= 0
    assert _abi.lib.dial_b200_kv4_attention_scratch_bytes(C.byref(sh), -1, 1, 1, 1, 0) == -1


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (16, 1), (40, 8), (1024, 1024)])
def test_scratch_of_every_size(q_heads, kv_heads):
    """Sizes at the ends of their ranges: never an arithmetic fault, none for a call
    that does nothing, and no less for a larger call than for a smaller one."""
    sh = kv4.make_shape(q_heads, kv_heads, 64, 640)
    size = kv4.attention_scratch_bytes
    for weights in (False, True):
        for seqs, rows, max_q, max_len in ((0, 5, 5, 99), (3, 0, 5, 99), (3, 5, 0, 99)):
            assert size(sh, seqs, rows, max_q, max_len, weights) == 0
        for seqs, rows, max_q in ((1, 1, 1), (7, 60, 9), (300, 300, 1), (300, 9000, 48), (65535, 65535, 1)):
            last = 0
            for max_len in (0, 1, 511, 1024, 1025, 4096, 70000, 1 << 20):
                got = size(sh, seqs, rows, max_q, max_len, weights)
                assert got >= last, (seqs, rows, max_q, max_len)
                last = got
        for max_len in (700, 1500, 40000):
            last = 0
            for q in (1, 2, 3, 4, 9, 10, 12, 13, 48, 49, 100, 1000):
                got = size(sh, 8, 8 * q, q, max_len, weights)
                assert got >= last, (q, max_len)
                last = got
            last = 0
            for seqs in (1, 2, 9, 100, 255, 256, 257, 600, 5000):
                got = size(sh, seqs, seqs, 1, max_len, weights)
                assert got >= last, (seqs, max_len)
                last = got


def test_scratch_of_refused_sizes():
    raw, ev = _abi.lib.dial_b200_kv4_attention_scratch_bytes, _abi.lib.dial_b200_kv4_evict_scratch_bytes
    for heads in ((17, 1), (64, 1), (30, 4), (0, 1), (4096, 2048)):
        assert raw(C.byref(kv4.make_shape(*heads, 64, 64)), 1, 1, 1, 64, 1) == -1
    sh = kv4.make_shape(32, 8, 64, 64)
    for sizes in ((65536, 1, 1, 64), (1, 1 << 27, 1, 64), (1, 1, 1 << 25, 64), (1, 1, 1, 1 << 31), (1, 1, 1, -1)):
        assert raw(C.byref(sh), *sizes, 0) == -1
    assert ev(C.byref(sh), 65536, 64, 8) == -1 and ev(C.byref(sh), 1, 64, -1) == -1
    with pytest.raises(dial_b200.DialError, match="exceeds the block table"):
        kv4._max_len(sh, 64 * 16 + 1)


def test_python_checks_name_the_tensor():
    c = Cache(1, 2, 64, 4, 2)
    cache, table = c.device("cpu")
    z = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4 * 128, dtype=torch.bfloat16)
    bad = dial_b200.DialError
    with pytest.raises(bad, match="CUDA device"):
        kv4.kv4_attention(c.sh, cache, q, table, z, z, 64)
    with pytest.raises(bad, match="^q: expected torch.bfloat16"):
        kv4.kv4_attention(c.sh, cache, q.half(), table, z, z, 64)
    with pytest.raises(bad, match="^lens"):
        kv4.kv4_attention(c.sh, cache, q, table, z, z.long(), 64)
    with pytest.raises(bad, match="^block_table"):
        kv4.kv4_attention(c.sh, cache, q, table[:, :2], z, z, 64)
    with pytest.raises(bad, match="^pages"):
        kv4.kv4_attention(c.sh, kv4.Kv4Cache(cache.pages[:1]), q, table, z, z, 64)
    with pytest.raises(bad, match="needs a cache with weights"):
        kv4.kv4_attention(c.sh, kv4.Kv4Cache(cache.pages), q, table, z, z, 64, accumulate=True)
    with pytest.raises(bad, match="^scratch"):
        kv4.kv4_evict(c.sh, cache, table, z, z, 64, 32, scratch=torch.zeros(4, dtype=torch.uint8))
    with pytest.raises(bad, match="^slots"):
        kv4.kv4_append(c.sh, cache, torch.zeros(3, 8 * 128, dtype=torch.bfloat16), table,
                       torch.zeros(3, dtype=torch.int32), z, z)
    with pytest.raises(bad, match="F16 or BF16"):
        kv4.make_shape(4, 2, 4, 4, dtype=torch.float32)
    with pytest.raises(bad, match="count -1"):
        kv4.kv4_read(c.sh, cache, table, z, z, -1)


def test_reference_codec():
    """The reference's rounding against torch's e4m3 and the e2m1 midpoints."""
    x = np.abs(np.random.default_rng(0).standard_normal(4000)) * 40
    want = torch.from_numpy(x.astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(E4M3[nearest(x.astype(np.float32).astype(np.float64), E4M3[:127])], want)
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 9.0, 0.2500001, 0.7499999]
    assert E2M1[nearest(np.array(mids), E2M1[:8])].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0.5, 0.5]
    r = np.random.default_rng(1).standard_normal((2, 3, 16, 128))
    k, ks = encode(r, 0.5)
    got = unpack(pack(k, ks, k, ks))
    np.testing.assert_array_equal(got[0], k)
    np.testing.assert_array_equal(got[3], ks)
    # half a step of e2m1 (2^-2 relative at most, 1/4 of the scale below 1) and
    # half a step of e4m3 on the largest (2^-4)
    d = np.abs(decode(k, ks, 0.5) - r).reshape(2, 3, 16, 8, 16)
    top = np.abs(r).reshape(2, 3, 16, 8, 16).max(-1, keepdims=True)
    assert (d <= top * (1 / 6 + 2 ** -4) * (1 + 2 ** -4)).all()
