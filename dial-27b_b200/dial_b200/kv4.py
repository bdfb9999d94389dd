"""4-bit KV cache: append, read back, attention and eviction (C ABI
dial_b200_kv4_*).

A paged cache in the NVFP4 form of the linears (e2m1 codes, an e4m3 scale for
every 16 dims): 144 bytes a token and kv head against 512 for the pages of
``attention_decode``.  A decode step is ``kv4_append`` (q/k RMSNorm, RoPE,
quantisation) and ``kv4_attention``; a prompt takes the same two calls with
more rows.  With ``accumulate`` the attention keeps each slot's summed weight,
by which ``kv4_evict`` cuts sessions that have reached their capacity.  The
reference's cache (llama3/cache.rs:9-265) holds the activation dtype and slides
instead.

Every op runs on the current stream of its tensors' device, allocates only its
results and, unless given, its scratch, and does not synchronise.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from ._abi import ACT_BF16, ACT_F16, DIAL_ERR_INVALID, DialError, Kv4Shape, call, lib

_ACT = {torch.bfloat16: ACT_BF16, torch.float16: ACT_F16}
_DTYPE = {ACT_BF16: torch.bfloat16, ACT_F16: torch.float16}
HEAD_DIM = 128
PAGE_TOKENS = 16
SLAB_BYTES = 2304


def make_shape(q_heads: int, kv_heads: int, max_blocks: int, num_blocks: int, max_pos: int = 0,
               eps: float = 1e-6, k_scale: float = 1.0, v_scale: float = 1.0,
               softmax_scale: float = 0.0, dtype: torch.dtype = torch.bfloat16) -> Kv4Shape:
    """max_pos: rows of the RoPE tables.  k_scale / v_scale stand beside the
    e4m3 scales: amax / 6 / k_scale of a 16-dim group should fall in [2^-6,
    448].  softmax_scale 0: 1 / sqrt(128)."""
    if dtype not in _ACT:
        raise DialError(DIAL_ERR_INVALID, f"activations must be F16 or BF16, got {dtype}")
    return Kv4Shape(q_heads, kv_heads, HEAD_DIM, max_blocks, num_blocks, max_pos, eps, k_scale,
                    v_scale, softmax_scale, _ACT[dtype])


@dataclass
class Kv4Cache:
    """pages uint8 [num_blocks, kv_heads, 2304]; weights f32 and positions
    int32 [num_blocks, kv_heads, 16] or None: what eviction ranks by."""
    pages: torch.Tensor
    weights: torch.Tensor | None = None
    positions: torch.Tensor | None = None

    @classmethod
    def empty(cls, sh: Kv4Shape, device, tracked: bool = False) -> "Kv4Cache":
        n, h = sh.num_blocks, sh.kv_heads
        z = lambda w, dt: torch.zeros(n, h, w, dtype=dt, device=device)  # noqa: E731
        return cls(z(SLAB_BYTES, torch.uint8),
                   z(PAGE_TOKENS, torch.float32) if tracked else None,
                   z(PAGE_TOKENS, torch.int32) if tracked else None)


def _bad(msg: str):
    raise DialError(DIAL_ERR_INVALID, msg)


def _need(name: str, t, dtype, shape, dev) -> int:
    """Address of a contiguous tensor of this dtype, shape and device (None in
    `shape`: any size); 0 for no tensor."""
    if t is None:
        return 0
    if t.dtype != dtype or t.device != dev or not t.is_contiguous() or t.dim() != len(shape) or any(
            w is not None and w != g for w, g in zip(shape, t.shape)):
        _bad(f"{name}: expected a contiguous {dtype} tensor {tuple(shape)} on {dev}, got {t.dtype} "
             f"{tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")
    return t.data_ptr()


def _rows(name: str, t, dtype, width: int, rows, dev) -> int:
    """Address of row-major rows of at least `width` elements, any row stride."""
    if (t.dtype != dtype or t.device != dev or t.dim() != 2 or t.shape[1] != width
            or (rows is not None and t.shape[0] != rows) or (t.shape[1] > 1 and t.stride(1) != 1)):
        _bad(f"{name}: expected {dtype} rows [{'rows' if rows is None else rows}, {width}] on {dev}, "
             f"got {t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}")
    return t.data_ptr()


def _ld(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _pool(sh: Kv4Shape, cache: Kv4Cache, dev):
    n, h = sh.num_blocks, sh.kv_heads
    return (_need("pages", cache.pages, torch.uint8, (n, h, SLAB_BYTES), dev),
            _need("weights", cache.weights, torch.float32, (n, h, PAGE_TOKENS), dev),
            _need("positions", cache.positions, torch.int32, (n, h, PAGE_TOKENS), dev))


def _launch(name: str, dev, *args):
    if dev.type != "cuda":
        _bad(f"{name}: tensors must be on a CUDA device, got {dev}")
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        call(name, *args, stream)
    else:
        with torch.cuda.device(dev):
            call(name, *args, stream)


def _scratch(given, nbytes: int, dev):
    if given is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    if given.device != dev or not given.is_contiguous() or given.numel() * given.element_size() < nbytes:
        _bad(f"scratch: expected {nbytes} contiguous bytes on {dev}")
    return given


def kv4_append(sh: Kv4Shape, cache: Kv4Cache, qkv, block_table, sids, slots, positions=None,
               q_norm_w=None, k_norm_w=None, cos=None, sin=None, q_out=None, want_q: bool = True):
    """Rows q | k | v into slots[m] of session sids[m] (a negative slot: a
    padding row), with RMSNorm if the norm weights are given and RoPE at
    positions[m] if cos and sin are; returns q after both [rows, q_heads * 128]
    (in q_out if given; None with want_q=False)."""
    dev, dt = qkv.device, _DTYPE[sh.act]
    width = (sh.q_heads + 2 * sh.kv_heads) * HEAD_DIM
    rows = qkv.shape[0]
    p_qkv = _rows("qkv", qkv, dt, width, None, dev)
    if q_out is None and want_q:
        q_out = torch.empty(rows, sh.q_heads * HEAD_DIM, dtype=dt, device=dev)
    p_q = _rows("q_out", q_out, dt, sh.q_heads * HEAD_DIM, rows, dev) if q_out is not None else 0
    i32 = torch.int32
    _launch("dial_b200_kv4_append", dev, C.byref(sh), p_qkv, _ld(qkv),
            _need("q_norm_w", q_norm_w, dt, (HEAD_DIM,), dev),
            _need("k_norm_w", k_norm_w, dt, (HEAD_DIM,), dev),
            _need("cos", cos, dt, (sh.max_pos, HEAD_DIM // 2), dev),
            _need("sin", sin, dt, (sh.max_pos, HEAD_DIM // 2), dev),
            *_pool(sh, cache, dev),
            _need("block_table", block_table, i32, (None, sh.max_blocks), dev),
            block_table.shape[0], _need("sids", sids, i32, (rows,), dev),
            _need("slots", slots, i32, (rows,), dev),
            _need("positions", positions, i32, (rows,), dev), p_q,
            _ld(q_out) if q_out is not None else 0, rows)
    return q_out


def kv4_read(sh: Kv4Shape, cache: Kv4Cache, block_table, sids, lens, count: int, first=None):
    """The values that slots first[i] + j (default j), j < count, of session
    sids[i] stand for: k and v [seqs, count, kv_heads, 128] in the activation
    dtype, zeros at and past lens[i]."""
    dev, i32 = sids.device, torch.int32
    n = sids.shape[0]
    if count < 0:
        _bad(f"count {count} is negative")
    k = torch.empty(n, count, sh.kv_heads, HEAD_DIM, dtype=_DTYPE[sh.act], device=dev)
    v = torch.empty_like(k)
    _launch("dial_b200_kv4_read", dev, C.byref(sh), _pool(sh, cache, dev)[0],
            _need("block_table", block_table, i32, (None, sh.max_blocks), dev),
            block_table.shape[0], _need("sids", sids, i32, (n,), dev),
            _need("first", first, i32, (n,), dev), _need("lens", lens, i32, (n,), dev), n, count,
            k.data_ptr(), v.data_ptr())
    return k, v


def attention_scratch_bytes(sh: Kv4Shape, seqs: int, rows: int, max_q: int, max_len: int,
                            accumulate: bool = False) -> int:
    return int(lib.dial_b200_kv4_attention_scratch_bytes(C.byref(sh), seqs, rows, max_q, max_len,
                                                         int(accumulate)))


def kv4_attention(sh: Kv4Shape, cache: Kv4Cache, q, block_table, sids, lens, max_len: int,
                  q_starts=None, max_q: int = 1, accumulate: bool = False, out=None, scratch=None):
    """Attention of q [rows, q_heads * 128] over the cached slots, causal at the
    end of each sequence: sequence i's queries are rows q_starts[i] ..
    q_starts[i + 1] - 1 (default: row i), the last of them sees slots 0 ..
    lens[i] - 1 of session sids[i].  max_q and max_len bound the queries and
    slots of a sequence.  accumulate adds each slot's probabilities to
    cache.weights.  Returns out [rows, q_heads * 128]."""
    dev, dt, i32 = q.device, _DTYPE[sh.act], torch.int32
    rows, n, width = q.shape[0], sids.shape[0], sh.q_heads * HEAD_DIM
    p_q = _rows("q", q, dt, width, None, dev)
    if out is None:
        # rows that no sequence names are left as they were: none here
        out = torch.empty(rows, width, dtype=dt, device=dev)
    p_out = _rows("out", out, dt, width, rows, dev)
    pages, weights, _ = _pool(sh, cache, dev)
    if accumulate and not weights:
        _bad("accumulate needs a cache with weights")
    buf = _scratch(scratch, attention_scratch_bytes(sh, n, rows, max_q, max_len, accumulate), dev)
    _launch("dial_b200_kv4_attention", dev, C.byref(sh), p_q, _ld(q), pages,
            weights if accumulate else 0,
            _need("block_table", block_table, i32, (None, sh.max_blocks), dev),
            block_table.shape[0], _need("sids", sids, i32, (n,), dev),
            _need("lens", lens, i32, (n,), dev), _need("q_starts", q_starts, i32, (n + 1,), dev), n,
            rows, max_q, max_len, p_out, _ld(out), buf.data_ptr() if buf is not None else 0)
    return out


def evict_scratch_bytes(sh: Kv4Shape, seqs: int, max_len: int, keep: int) -> int:
    return int(lib.dial_b200_kv4_evict_scratch_bytes(C.byref(sh), seqs, max_len, keep))


def kv4_evict(sh: Kv4Shape, cache: Kv4Cache, block_table, sids, lens, max_len: int, keep: int,
              recent: int = 0, dst_table=None, lens_out=None, scratch=None):
    """Cut the sessions to their `keep` most attended entries, kv head by kv
    head; entries newer than (newest position - recent) come first.  In place,
    or into the pages of dst_table.  Returns the new lengths [seqs]."""
    dev, i32 = sids.device, torch.int32
    n = sids.shape[0]
    pages, weights, positions = _pool(sh, cache, dev)
    if lens_out is None:
        lens_out = torch.empty(n, dtype=i32, device=dev)
    sessions = block_table.shape[0]
    if keep < 0 or max_len < 0:
        _bad(f"keep {keep} / max_len {max_len} is negative")
    buf = _scratch(scratch, evict_scratch_bytes(sh, n, max_len, keep), dev)
    _launch("dial_b200_kv4_evict", dev, C.byref(sh), pages, weights, positions,
            _need("block_table", block_table, i32, (None, sh.max_blocks), dev),
            _need("dst_table", dst_table, i32, (sessions, sh.max_blocks), dev), sessions,
            _need("sids", sids, i32, (n,), dev), _need("lens", lens, i32, (n,), dev),
            _need("lens_out", lens_out, i32, (n,), dev), n, max_len, keep, recent,
            buf.data_ptr() if buf is not None else 0)
    return lens_out
