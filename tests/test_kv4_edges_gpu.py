"""The 4-bit KV cache operators at the edges of what they accept: scratch on
every boundary that is allowed, queries that are not finite or near the ends of
their range, probabilities far below the largest, sizes that take the rarer
paths.  References as in kv4_case.py."""

import numpy as np
import pytest
import torch

from kv4_case import DIM, Cache, act_round, i32, norm_rope, same_slabs
from test_kv4_gpu import check_attention

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


# ------------------------------------------------- queries that are not finite
@pytest.mark.parametrize("lens,queries", [((40, 33), (5, 2)), ((2600, 90), (200, 90)), ((2600, 1500), (1, 5)),
                                          ((300, 20), (60, 17)), ((1100, 1024), (12, 1))])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_queries_of_nan_and_infinity(cuda, lens, queries, dt):
    """A query head with a NaN gives NaN wherever it sees a slot, whole or cut over
    the GPU, in out and in the weights of the slots it sees; one with an infinity
    NaN in out; neither reaches another query, head, or a slot it does not see."""
    from dial_b200 import kv4

    c = Cache(62, 2, max(lens), 8, 2, dt=dt)
    cache, table = c.device(cuda)
    q = torch.randn(sum(queries), 8 * DIM, device=cuda).to(dt)
    clean = host(q)
    bad = [(0, 1, float("nan")), (queries[0] - 1, 6, float("nan")), (sum(queries) - 1, 3, float("inf")),
           (sum(queries) - 1, 4, float("-inf"))]
    want = np.zeros((sum(queries), 8), bool)
    for row, head, value in bad:
        q[row, head * DIM + 5] = value
        want[row, head] = True
    before = host(cache.weights)
    out = kv4.kv4_attention(c.sh, cache, q, table, i32(cuda, 0, 1), i32(cuda, *lens), max(lens),
                            q_starts=i32(cuda, 0, queries[0], sum(queries)), max_q=max(queries),
                            accumulate=True)
    out, w = host(out).reshape(-1, 8, DIM), host(cache.weights)
    np.testing.assert_array_equal(np.isnan(out), np.broadcast_to(want[..., None], out.shape))
    at = 0
    for s, (n, m) in enumerate(zip(lens, queries)):
        o, b, sums, sb = c.attend(clean[at:at + m], s, n)
        fine = ~want[at:at + m]
        d = np.abs(out[at:at + m] - o.reshape(m, 8, DIM))[fine]
        assert (d <= b.reshape(m, 8, DIM)[fine]).all()
        if s == 0:
            nan = np.zeros((n, 2), bool)
            for row, head, value in bad[:2]:
                nan[:max(0, n - m + 1 + row), head // 4] = True
            blk, off = c.at(0, n)
            got, old = w[blk, :, off], before[blk, :, off]
            np.testing.assert_array_equal(np.isnan(got), nan)
            d, lim = np.abs(got - old - sums), sb + 2.0 ** -23 * (2 * np.abs(old) + sums)
            assert (d <= lim)[~nan].all()
        at += m


# ---------------------------------------------------------- ends of the range
@pytest.mark.parametrize("power", [100, 116, 125, -110])
@pytest.mark.parametrize("queries,n", [(1, 900), (5, 1300), (70, 700)])
def test_queries_near_the_ends_of_bf16(cuda, power, queries, n):
    """Finite queries up to 2^127 and down to 2^-112, with a softmax scale that brings
    their scores back: as for ordinary ones."""
    from dial_b200 import kv4

    c = Cache(63, 1, n, 8, 2)
    scale = float(np.float32(2.0 ** (-power if power > 0 else 99) * DIM ** -0.5))
    sh = kv4.make_shape(8, 2, c.max_blocks, c.pages.shape[0], k_scale=c.k_scale, v_scale=c.v_scale,
                        softmax_scale=scale)
    cache, table = c.device(cuda)
    q = (torch.randn(queries, 8 * DIM, device=cuda).clamp(-3.9, 3.9).double() * 2.0 ** power).to(BF16)
    before = host(cache.weights)
    out = kv4.kv4_attention(sh, cache, q, table, i32(cuda, 0), i32(cuda, n), n, q_starts=i32(cuda, 0, queries),
                            max_q=queries, accumulate=True)
    o, b, s, sb = c.attend(host(q), 0, n, scale)
    assert np.isfinite(b).all() and (np.abs(host(out) - o) <= b).all()
    blk, off = c.at(0, n)
    d = np.abs(host(cache.weights)[blk, :, off] - before[blk, :, off] - s)
    assert (d <= sb + 2.0 ** -23 * (2 * before[blk, :, off] + s)).all()


@pytest.mark.parametrize("power", [14, 19, 22, 24, 25, 26, 27, 28, 30, 40, 80, 120])
@pytest.mark.parametrize("queries,n", [(1, 900), (1, 3000), (5, 1300), (70, 700)])
def test_scores_far_beyond_f32s_whole_numbers(cuda, power, queries, n):
    """Queries of 2^power under the ordinary scale: a head takes its best slot's values
    and adds 1 to its weight wherever the runner-up is further off than the roundings of
    32-bit scores (2^-18 of sum |q k|, twice attend's bound) and than 40; where it is
    not, the result lies between the values.  f16 probabilities cost 2^-11, the output
    half a step; the weight of a lone slot is 1 but for 2^-20 (exponentials and 1 / l)."""
    from dial_b200 import kv4

    c = Cache(71, 2, n, 8, 2)
    cache, table = c.device(cuda)
    q = (torch.randn(queries + 1, 8 * DIM, device=cuda).clamp(-3.9, 3.9).double() * 2.0 ** power).to(BF16)
    before = host(cache.weights)
    out = host(kv4.kv4_attention(c.sh, cache, q, table, i32(cuda, 1, 0), i32(cuda, n, 77), n,
                                 q_starts=i32(cuda, 0, queries, queries + 1), max_q=queries,
                                 accumulate=True)).reshape(queries + 1, 8, DIM)
    assert np.isfinite(out).all()
    added, decided = host(cache.weights) - before, 0
    for sid, rows, length in ((1, range(queries), n), (0, [queries], 77)):
        K, V = c.values(sid, length)
        Q = host(q).reshape(-1, 8, DIM)
        want, open_ = np.zeros((length, 2)), np.zeros(2)
        for j in rows:
            seen = length - len(rows) + 1 + j - rows[0]
            for h in range(8):
                k, v = K[:seen, h // 4], V[:seen, h // 4]
                s = (k @ Q[j, h]) * DIM ** -0.5
                best = int(s.argmax())
                gap = s[best] - np.delete(s, best).max()
                noise = 2.0 ** -18 * (np.abs(k) @ np.abs(Q[j, h])).max() * DIM ** -0.5
                if gap > max(noise, 40.0):
                    decided += 1
                    want[best, h // 4] += 1
                    d = np.abs(out[j, h] - v[best])
                    assert (d <= (2.0 ** -11 + 2.0 ** -8) * np.abs(v[best]) + 2.0 ** -30).all()
                else:
                    open_[h // 4] += 1
                    eps = 2.0 ** -7 * np.abs(v).max()
                    assert (out[j, h] >= v.min(0) - eps).all() and (out[j, h] <= v.max(0) + eps).all()
        blk, off = c.at(sid, length)
        d = added[blk, :, off] - want
        lim = 2.0 ** -20 * want + 2.0 ** -22 * (before[blk, :, off] + want)
        assert (d >= -lim).all() and (d <= lim + open_ * (1 + 2.0 ** -10)).all()
    assert decided > 0.8 * 8 * (queries + 1) or power < 19


@pytest.mark.parametrize("queries", [3, 60])
def test_scales_that_leave_nothing_of_a_score(cuda, queries):
    """Zero queries and ordinary ones under a scale of 1e-30: every slot that a query
    sees has the same weight, the others none."""
    from dial_b200 import kv4

    c = Cache(64, 1, 200, 8, 2)
    sh = kv4.make_shape(8, 2, c.max_blocks, c.pages.shape[0], k_scale=c.k_scale, v_scale=c.v_scale,
                        softmax_scale=1e-30)
    cache, table = c.device(cuda)
    q = torch.randn(queries, 8 * DIM, device=cuda).to(BF16)
    q[1] = 0
    before = host(cache.weights)
    out = kv4.kv4_attention(sh, cache, q, table, i32(cuda, 0), i32(cuda, 200), 200,
                            q_starts=i32(cuda, 0, queries), max_q=queries, accumulate=True)
    o, b, s, sb = c.attend(host(q), 0, 200, float(np.float32(1e-30)))
    assert (np.abs(host(out) - o) <= b).all()
    blk, off = c.at(0, 200)
    d = np.abs(host(cache.weights)[blk, :, off] - before[blk, :, off] - s)
    assert (d <= sb + 2.0 ** -23 * (2 * before[blk, :, off] + s)).all()


# ------------------------------------------------------- items of one tile
def test_items_without_blocks_in_a_tile(cuda):
    """Sequences of one tile of rows, of two, and of two of which the first sees no
    slot, in turn and several to a CTA: each item's results go to its own rows."""
    from dial_b200 import kv4

    c = Cache(66, 40, 502, 32, 8)
    seqs = [((330, 33), (270, 14), (20, 60), (499, 17))[i % 4] for i in range(40)]
    seqs = [(n + i % 4, m) for i, (n, m) in enumerate(seqs)]
    cache, table = c.device(cuda)
    starts = np.cumsum([0] + [m for _, m in seqs])
    q = torch.randn(int(starts[-1]), 32 * DIM, device=cuda).to(BF16)
    before = host(cache.weights)
    out = host(kv4.kv4_attention(c.sh, cache, q, table, torch.arange(40, dtype=torch.int32, device=cuda),
                                 i32(cuda, *[n for n, _ in seqs]), 502, q_starts=i32(cuda, *starts.tolist()),
                                 max_q=60, accumulate=True))
    w = host(cache.weights)
    for i, (n, m) in enumerate(seqs):
        o, b, s, sb = c.attend(host(q[starts[i]:starts[i + 1]]), i, n)
        assert (np.abs(out[starts[i]:starts[i + 1]] - o) <= b).all(), i
        blk, off = c.at(i, n)
        d = np.abs(w[blk, :, off] - before[blk, :, off] - s)
        assert (d <= sb + 2.0 ** -23 * (2 * before[blk, :, off] + s)).all(), i


# ------------------------------------------------------------ long flat tails
@pytest.mark.parametrize("sessions,n,heads,queries,tops", [(37, 1 << 20, (8, 8), 1, 8),
                                                           (1, 1 << 17, (64, 8), 608, 1)])
def test_a_long_tail_far_below_the_largest(cuda, sessions, n, heads, queries, tops):
    """`tops` slots share the largest score (one for each warp that takes a share of a
    sequence) and all others lie 2^-25.1 of it below: their sum counts, 0.4 % here,
    whatever the length.  Values are -a for the first and a for the others, so that
    out = a (T - 1) / (T + 1) with T the tail's sum.  Bound, on a (T + 1) / (T + 1) = a: f16
    probabilities 2^-11; f32 sums: a warp or row takes 2^17 slots, 16 a step of the
    product, each of the 2^13 partial sums off by 2^-23 at most (truncated), 2^-10, and l by
    2^13 additions rounded to 2^-24, 2^-11; half a step of f16, 2^-11.  All sessions
    read the same three pages."""
    from dial_b200 import kv4
    from kv4_case import PAGE, pack

    q_heads, H = heads
    blocks = n // PAGE
    sh = kv4.make_shape(q_heads, H, blocks, 4, k_scale=0.5, v_scale=0.0625, softmax_scale=1.0, dtype=F16)
    one = np.full((3, H, PAGE, 8), 0x38, np.uint8)  # scale 1
    k = np.zeros((3, H, PAGE, DIM), np.uint8)
    v = np.full((3, H, PAGE, DIM), 7, np.uint8)     # +6
    k[1, :, 5, 0] = 7
    v[1, :, 5] = 15                                 # -6
    pages = np.zeros((4, H, 2304), np.uint8)
    pages[:3] = pack(k, one, v, one)
    table = torch.zeros(sessions, blocks, dtype=torch.int32, device=cuda)
    table[:, :tops] = 1
    cache = kv4.Kv4Cache(torch.from_numpy(pages).to(cuda))
    t = np.float64(np.float16(25.1 * np.log(2) / 3))
    q = torch.zeros(sessions * queries, q_heads, DIM, dtype=F16, device=cuda)
    q[..., 0] = float(t)
    out = kv4.kv4_attention(sh, cache, q.reshape(-1, q_heads * DIM), table,
                            torch.arange(sessions, dtype=torch.int32, device=cuda),
                            torch.full((sessions,), n, dtype=torch.int32, device=cuda), n,
                            q_starts=i32(cuda, *range(0, sessions * queries + 1, queries)), max_q=queries)
    seen = np.tile(n - queries + 1 + np.arange(queries), sessions)
    tail = (seen - tops) * np.exp(-3 * t) / tops
    a = 6 * 0.0625
    want = (a * (tail - 1) / (tail + 1))[:, None]
    assert tail.min() > 0.0035
    d = np.abs(host(out) - want)
    bound = a * (2.0 ** -11 + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -11)
    assert (d <= bound).all(), (d.max(), bound)


def test_a_large_score_in_the_second_half_of_a_block(cuda):
    """A block of 128 keys whose first 64 score 7.5 above the keys before (base 2) and
    whose second half holds one of 27: the 64 add 2^-13.5 to its weight, twelve
    times that to the values here.  Bound: half a step of f16, and 2^-16 of the largest value
    for the rest: scores of 27 off by 2^-18.6 (the f32 scale and the exponential), sums
    of 300 terms; probabilities in f16 are off by 2^-11 of that 2^-13.5.  Sessions
    enough, all on the same pages, that CTAs take whole items."""
    from dial_b200 import kv4

    n, queries, sessions = 316, 60, 40
    c = Cache(67, 1, n, 8, 8, dt=F16)
    score = np.zeros(n)
    score[128:192], score[192:256], score[222], score[256:] = 7.5, -39.0, 27.0, -39.0
    for slot in range(n):
        k, v = np.zeros((8, DIM)), np.full((8, DIM), 2.0 ** -5)
        k[:, 0] = score[slot]
        if 128 <= slot < 192:
            v[:] = 0.375
        c.put(0, slot, k, v, 0)
    assert np.array_equal(c.values(0, n)[0][:, 7, 0], score)
    sh = kv4.make_shape(8, 8, c.max_blocks, c.pages.shape[0], k_scale=c.k_scale, v_scale=c.v_scale,
                        softmax_scale=float(np.float32(np.log(2))), dtype=F16)
    cache, table = c.device(cuda)
    q = torch.zeros(sessions * queries, 8 * DIM, dtype=F16, device=cuda)
    q[:, ::DIM] = 1
    out = host(kv4.kv4_attention(sh, cache, q, table.expand(sessions, -1).contiguous(),
                                 torch.arange(sessions, dtype=torch.int32, device=cuda),
                                 i32(cuda, *[n] * sessions), n,
                                 q_starts=i32(cuda, *range(0, sessions * queries + 1, queries)),
                                 max_q=queries)).reshape(sessions, queries, -1)
    want = c.attend(host(q[:queries]), 0, n, float(np.float32(np.log(2))))[0]
    d = np.abs(out - want)
    assert (d <= 2.0 ** -11 * np.abs(want) + 2.0 ** -16 * 0.375).all(), d.max()


# -------------------------------------------------------------- bad sequences
def test_read_leaves_bad_sessions_out(cuda):
    """Sequences of no session: reported, and their rows stay as they were, those past
    their length among them."""
    import ctypes as C

    import dial_b200
    from dial_b200 import _abi

    c = Cache(65, 2, 64, 4, 2)
    cache, table = c.device(cuda)
    k = torch.full((4, 5, 2, DIM), 3.0, dtype=BF16, device=cuda)
    v = torch.full_like(k, 4.0)
    sids, lens = i32(cuda, 1, 2, -1, 0), i32(cuda, 3, 2, 0, 64)
    _abi.call("dial_b200_kv4_read", C.byref(c.sh), cache.pages.data_ptr(), table.data_ptr(), 2, sids.data_ptr(),
              None, lens.data_ptr(), 4, 5, k.data_ptr(), v.data_ptr(),
              torch.cuda.current_stream(cuda).cuda_stream)
    torch.cuda.synchronize()
    assert dial_b200.device_status(clear=True) == 0x104
    assert (k[1:3] == 3.0).all() and (v[1:3] == 4.0).all()
    assert (k[0, 3:] == 0).all() and (v[0, 3:] == 0).all()
    for i, (sid, n) in ((0, (1, 3)), (3, (0, 5))):
        kk, vv = c.values(sid, n)
        want = torch.from_numpy(kk.astype(np.float32)).to(BF16)
        assert torch.equal(k[i, :n].cpu(), want)
        assert torch.equal(v[i, :n].cpu(), torch.from_numpy(vv.astype(np.float32)).to(BF16))


# -------------------------------------------------------------- arguments
def test_single_queries_take_no_max_q(cuda):
    """Without q_starts, max_q is not looked at."""
    from dial_b200 import kv4

    c = Cache(68, 2, 1200, 8, 2)
    cache, table = c.device(cuda)
    q = torch.randn(2, 8 * DIM, device=cuda).to(BF16)
    args = (c.sh, cache, q, table, i32(cuda, 0, 1), i32(cuda, 1200, 37), 1200)
    want = kv4.kv4_attention(*args)
    for max_q in (0, 9, 100):
        out = torch.full_like(q, 5.0)
        assert torch.equal(kv4.kv4_attention(*args, max_q=max_q, out=out), want)


# ------------------------------------------------------------ the rarer paths
@pytest.mark.parametrize("n,queries,heads,dt", [
    (1200, 1100, (8, 1), BF16),   # 69 tiles of rows: items of three chunks, 35 pairs of tiles
    (3000, 700, (16, 2), F16),    # 44 tiles over twelve key blocks, as few see the last
    (700, 40, (16, 1), F16), (300, 300, (16, 1), BF16),  # 16 heads a group
    (900, 130, (8, 2), F16)])
def test_prompts_with_weights(cuda, n, queries, heads, dt):
    c = Cache(69, 3, n, *heads, dt=dt)
    check_attention(c, cuda, [(2, n, queries), (0, min(n, 77), 5), (1, 33, 20)], spare_rows=1)


@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_of_a_session_past_shared_memory(cuda, out_of_place):
    """More slots than a CTA keeps the keys of (24576), weights with many ties."""
    from dial_b200 import kv4

    n, keep, recent = 25003, 9001, 500
    c = Cache(70, 1, n, 2, 2)
    b, o = c.at(0, n)
    for h in range(2):
        c.positions[b, h, o] = np.cumsum(c.rng.integers(1, 3, n))
    c.weights = np.round(c.weights * 8).astype(np.float32)
    dst = c.table.copy()
    if out_of_place:
        kb, first = -(-keep // 16), c.sh.num_blocks
        for x in ("pages", "weights", "positions"):
            a = getattr(c, x)
            setattr(c, x, np.concatenate([a, a[:1].repeat(kb, 0)]))
        c.sh.num_blocks = first + kb
        dst[:] = -1
        dst[0, :kb] = np.arange(first, first + kb)
    cache, table = c.device(cuda)
    new = kv4.kv4_evict(c.sh, cache, table, i32(cuda, 0), i32(cuda, n), n, keep, recent,
                        dst_table=torch.from_numpy(dst).to(cuda) if out_of_place else None)
    assert host(new).tolist() == [c.evict(0, n, keep, recent, dst)]
    np.testing.assert_array_equal(host(cache.pages), c.pages)
    np.testing.assert_array_equal(host(cache.weights), c.weights)
    np.testing.assert_array_equal(host(cache.positions), c.positions)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_append_of_rows_at_the_ends_of_the_type(cuda, dt):
    """Heads of values near the type's largest and smallest, of one value beside zeros, and
    of zeros alone, with norm and RoPE: q and the slabs equal the reference."""
    from dial_b200 import kv4

    c = Cache(72, 1, 64, 6, 2, dt=dt, fill=False, max_pos=300)
    cache, table = c.device(cuda)
    rows = 40
    lo, hi = (-14, 14) if dt == F16 else (-126, 125)
    x = c.rng.standard_normal((rows, 10, DIM)).clip(-3.5, 3.5)
    x *= 2.0 ** c.rng.integers(lo, hi + 1, (rows, 10, 1))
    x[0] = 0
    x[1, :, 1:] = 0
    x[2, :, ::2] *= 2.0 ** -9
    x = act_round(x.reshape(rows, -1), dt)
    slots = np.arange(rows, dtype=np.int32)
    pos = (slots * 7).astype(np.int32)
    tab = np.arange(300)[:, None] * 1e6 ** (-np.arange(64) / 64)
    cos, sin = (act_round(f(tab), dt) for f in (np.cos, np.sin))
    w = act_round(1 + 0.2 * c.rng.standard_normal(DIM), dt)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda).to(dt)  # noqa: E731
    q = kv4.kv4_append(c.sh, cache, t(x), table, i32(cuda, *[0] * rows), i32(cuda, *slots.tolist()),
                       i32(cuda, *pos.tolist()), t(w), t(w), t(cos), t(sin))
    hd = x.reshape(rows, -1, DIM)
    eps = float(np.float32(1e-6))
    qr = norm_rope(hd[:, :6], w, cos[pos], sin[pos], eps, dt)
    kr = norm_rope(hd[:, 6:8], w, cos[pos], sin[pos], eps, dt)
    np.testing.assert_array_equal(host(q), qr.reshape(rows, -1))
    for m in range(rows):
        c.put(0, m, kr[m], hd[m, 8:], pos[m])
    same_slabs(host(cache.pages), c.pages)
