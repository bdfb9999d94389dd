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
results and, unless given, its scratch, and does not synchronise.  A call
captured into a graph keeps the scratch it was given (or allocated from the
capture's pool): two graphs that may run at the same time need two.
"""

from __future__ import annotations

import ctypes as C
import functools
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


def _need(name: str, t, dtype, numel: int, idx: int) -> int:
    """Address of a contiguous tensor of this dtype and size on device `idx`; 0 for
    no tensor."""
    if t is None:
        return 0
    if t.dtype is dtype and t.numel() == numel and t.is_contiguous() and t.get_device() == idx:
        return t.data_ptr()
    _bad(f"{name}: expected a contiguous {dtype} tensor of {numel} elements on device {idx}, got "
         f"{t.dtype} {tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")


def _table(name: str, t, width: int, idx: int):
    """Address and rows of a block table [sessions, width]."""
    if (t.dtype is torch.int32 and t.dim() == 2 and t.size(1) == width and t.is_contiguous()
            and t.get_device() == idx):
        return t.data_ptr(), t.size(0)
    _bad(f"{name}: expected a contiguous int32 tensor [sessions, {width}] on device {idx}, got "
         f"{t.dtype} {tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")


def _rows(name: str, t, dtype, rows, width: int, idx: int):
    """Address and row stride of rows of `width` elements (rows None: any number)."""
    if (t.dtype is dtype and t.dim() == 2 and t.size(1) == width
            and (rows is None or t.size(0) == rows) and t.stride(1) == 1
            and t.get_device() == idx):
        return t.data_ptr(), t.stride(0) if t.size(0) > 1 else width
    _bad(f"{name}: expected {dtype} rows [{'rows' if rows is None else rows}, {width}] on device {idx}, "
         f"got {t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}")


def _max_len(sh: Kv4Shape, max_len: int):
    if not 0 <= max_len <= PAGE_TOKENS * sh.max_blocks:
        _bad(f"max_len {max_len} exceeds the block table's {PAGE_TOKENS * sh.max_blocks} slots")


def _launch(name: str, idx: int, *args):
    """The call on the current stream of device `idx`, which is made current."""
    if idx < 0:
        _bad(f"{name}: tensors must be on a CUDA device")
    stream = _raw_stream(idx)
    if _current_device() == idx:
        call(name, *args, stream)
    else:
        with torch.cuda.device(idx):
            call(name, *args, stream)


def _raw_stream(idx: int) -> int:
    return torch._C._cuda_getCurrentRawStream(idx)


def _current_device() -> int:
    return torch._C._cuda_getDevice()


def _scratch(given, nbytes: int, like):
    """Address of the scratch, and what keeps it alive during the call."""
    if given is None:
        if nbytes <= 0:  # none is needed, or the call refuses its sizes
            return 0, None
        given = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    elif (given.get_device() != like.get_device() or not given.is_contiguous()
          or given.numel() * given.element_size() < nbytes):
        _bad(f"scratch: expected {nbytes} contiguous bytes on {like.device}")
    return given.data_ptr(), given


def kv4_append(sh: Kv4Shape, cache: Kv4Cache, qkv, block_table, sids, slots, positions=None,
               q_norm_w=None, k_norm_w=None, cos=None, sin=None, q_out=None, want_q: bool = True):
    """Rows q | k | v into slots[m] of session sids[m] (a negative slot: a
    padding row), with RMSNorm if the norm weights are given and RoPE at
    positions[m] if cos and sin are; returns q after both [rows, q_heads * 128]
    (in q_out if given; None with want_q=False)."""
    idx, dt, i32 = qkv.get_device(), _DTYPE[sh.act], torch.int32
    H, Q, nb = sh.kv_heads, sh.q_heads, sh.num_blocks
    rows = qkv.size(0)
    p_qkv, ld = _rows("qkv", qkv, dt, None, (Q + 2 * H) * HEAD_DIM, idx)
    p_q = ld_q = 0
    if q_out is not None:
        p_q, ld_q = _rows("q_out", q_out, dt, rows, Q * HEAD_DIM, idx)
    elif want_q:
        q_out = torch.empty(rows, Q * HEAD_DIM, dtype=dt, device=qkv.device)
        p_q, ld_q = q_out.data_ptr(), Q * HEAD_DIM
    p_bt, sessions = _table("block_table", block_table, sh.max_blocks, idx)
    slabs, rope = nb * H, sh.max_pos * (HEAD_DIM // 2)
    _launch("dial_b200_kv4_append", idx, C.byref(sh), p_qkv, ld,
            _need("q_norm_w", q_norm_w, dt, HEAD_DIM, idx),
            _need("k_norm_w", k_norm_w, dt, HEAD_DIM, idx),
            _need("cos", cos, dt, rope, idx), _need("sin", sin, dt, rope, idx),
            _need("pages", cache.pages, torch.uint8, slabs * SLAB_BYTES, idx),
            _need("weights", cache.weights, torch.float32, slabs * PAGE_TOKENS, idx),
            _need("positions pool", cache.positions, i32, slabs * PAGE_TOKENS, idx), p_bt, sessions,
            _need("sids", sids, i32, rows, idx), _need("slots", slots, i32, rows, idx),
            _need("positions", positions, i32, rows, idx), p_q, ld_q, rows)
    return q_out


def kv4_read(sh: Kv4Shape, cache: Kv4Cache, block_table, sids, lens, count: int, first=None):
    """The values that slots first[i] + j (default j), j < count, of session
    sids[i] stand for: k and v [seqs, count, kv_heads, 128] in the activation
    dtype, zeros at and past lens[i]."""
    idx, i32, H = sids.get_device(), torch.int32, sh.kv_heads
    n = sids.numel()
    if count < 0:
        _bad(f"count {count} is negative")
    k = torch.empty(n, count, H, HEAD_DIM, dtype=_DTYPE[sh.act], device=sids.device)
    v = torch.empty_like(k)
    p_bt, sessions = _table("block_table", block_table, sh.max_blocks, idx)
    _launch("dial_b200_kv4_read", idx, C.byref(sh),
            _need("pages", cache.pages, torch.uint8, sh.num_blocks * H * SLAB_BYTES, idx), p_bt,
            sessions, _need("sids", sids, i32, n, idx), _need("first", first, i32, n, idx),
            _need("lens", lens, i32, n, idx), n, count, k.data_ptr(), v.data_ptr())
    return k, v


def attention_scratch_bytes(sh: Kv4Shape, seqs: int, rows: int, max_q: int, max_len: int,
                            accumulate: bool = False) -> int:
    return _attention_scratch(sh.q_heads, sh.kv_heads, seqs, rows, max_q, max_len, bool(accumulate))


@functools.lru_cache(maxsize=1024)
def _attention_scratch(q_heads, kv_heads, seqs, rows, max_q, max_len, accumulate) -> int:
    sh = make_shape(q_heads, kv_heads, 1, 1)  # the size goes by the heads alone
    return int(lib.dial_b200_kv4_attention_scratch_bytes(C.byref(sh), seqs, rows, max_q, max_len,
                                                         int(accumulate)))


def kv4_attention(sh: Kv4Shape, cache: Kv4Cache, q, block_table, sids, lens, max_len: int,
                  q_starts=None, max_q: int = 1, accumulate: bool = False, out=None, scratch=None):
    """Attention of q [rows, q_heads * 128] over the cached slots, causal at the
    end of each sequence: sequence i's queries are rows q_starts[i] ..
    q_starts[i + 1] - 1 (default: row i), the last of them sees slots 0 ..
    lens[i] - 1 of session sids[i].  max_q (with q_starts) and max_len bound the
    queries and slots of a sequence.  accumulate adds each slot's probabilities to
    cache.weights.  Returns out [rows, q_heads * 128]."""
    idx, dt, i32 = q.get_device(), _DTYPE[sh.act], torch.int32
    H, rows, n, width = sh.kv_heads, q.size(0), sids.numel(), sh.q_heads * HEAD_DIM
    slabs = sh.num_blocks * H
    p_q, ld = _rows("q", q, dt, None, width, idx)
    if out is None:
        out = torch.empty(rows, width, dtype=dt, device=q.device)
        p_out, ld_out = out.data_ptr(), width
    else:
        p_out, ld_out = _rows("out", out, dt, rows, width, idx)
    p_w = 0
    if accumulate:
        p_w = _need("weights", cache.weights, torch.float32, slabs * PAGE_TOKENS, idx)
        if not p_w:
            _bad("accumulate needs a cache with weights")
    p_bt, sessions = _table("block_table", block_table, sh.max_blocks, idx)
    _max_len(sh, max_len)
    if q_starts is None:
        max_q = 1
    p_s, keep = _scratch(scratch, attention_scratch_bytes(sh, n, rows, max_q, max_len, accumulate), q)
    _launch("dial_b200_kv4_attention", idx, C.byref(sh), p_q, ld,
            _need("pages", cache.pages, torch.uint8, slabs * SLAB_BYTES, idx), p_w, p_bt,
            sessions, _need("sids", sids, i32, n, idx), _need("lens", lens, i32, n, idx),
            _need("q_starts", q_starts, i32, n + 1, idx), n, rows, max_q, max_len, p_out, ld_out, p_s)
    return out


def evict_scratch_bytes(sh: Kv4Shape, seqs: int, max_len: int, keep: int) -> int:
    return _evict_scratch(sh.kv_heads, seqs, max_len, keep)


@functools.lru_cache(maxsize=1024)
def _evict_scratch(kv_heads, seqs, max_len, keep) -> int:
    sh = make_shape(kv_heads, kv_heads, 1, 1)
    return int(lib.dial_b200_kv4_evict_scratch_bytes(C.byref(sh), seqs, max_len, keep))


def kv4_evict(sh: Kv4Shape, cache: Kv4Cache, block_table, sids, lens, max_len: int, keep: int,
              recent: int = 0, dst_table=None, lens_out=None, scratch=None):
    """Cut the sessions to their `keep` most attended entries, kv head by kv
    head; entries newer than (newest position - recent) come first.  In place,
    or into the pages of dst_table.  Returns the new lengths [seqs]."""
    idx, i32, H, nb = sids.get_device(), torch.int32, sh.kv_heads, sh.num_blocks
    n, slots = sids.numel(), nb * H * PAGE_TOKENS
    if keep < 0:
        _bad(f"keep {keep} is negative")
    _max_len(sh, max_len)
    if lens_out is None:
        lens_out = torch.empty(n, dtype=i32, device=sids.device)
    p_bt, sessions = _table("block_table", block_table, sh.max_blocks, idx)
    p_s, alive = _scratch(scratch, evict_scratch_bytes(sh, n, max_len, keep), sids)
    _launch("dial_b200_kv4_evict", idx, C.byref(sh),
            _need("pages", cache.pages, torch.uint8, nb * H * SLAB_BYTES, idx),
            _need("weights", cache.weights, torch.float32, slots, idx),
            _need("positions pool", cache.positions, i32, slots, idx), p_bt,
            _need("dst_table", dst_table, i32, sessions * sh.max_blocks, idx), sessions,
            _need("sids", sids, i32, n, idx), _need("lens", lens, i32, n, idx),
            _need("lens_out", lens_out, i32, n, idx), n, max_len, keep, recent, p_s)
    return lens_out
