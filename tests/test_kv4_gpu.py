"""The 4-bit KV cache operators against a plain 64-bit reference (kv4_case.py):
codes, scales, read-back values and evictions equal it; attention is within the
bound that the reference derives from the roundings."""

import numpy as np
import pytest
import torch

from kv4_case import DIM, PAGE, Cache, act_round, decode, encode, i32, norm_rope, same_slabs

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def clear_status(cuda):
    import dial_b200

    dial_b200.device_status(clear=True)


def host(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def check_attention(c, cuda, seqs, max_q=None, max_len=None, weights=True, q_scale=1.5, spare_rows=0,
                    stride=0, dev=None, scratch=None):
    """Run kv4_attention for seqs = [(sid, len, queries)] and compare out and
    the running weights with the reference; returns the device cache."""
    from dial_b200 import kv4

    counts = [n for _, _, n in seqs]
    rows = sum(counts) + spare_rows
    q = act_round(c.rng.standard_normal((rows, c.QH * DIM)) * q_scale, c.dt)
    cache, table = dev if dev else c.device(cuda)
    qd = torch.zeros(rows, c.QH * DIM + stride, dtype=c.dt, device=cuda)
    qd[:, :c.QH * DIM] = torch.from_numpy(q).to(cuda)
    out = torch.full((rows, c.QH * DIM + stride), 7.0, dtype=c.dt, device=cuda)
    starts = None if counts == [1] * len(counts) and not spare_rows else i32(
        cuda, *([0] + np.cumsum(counts).tolist()))
    before = host(cache.weights)
    kv4.kv4_attention(c.sh, cache, qd[:, :c.QH * DIM], table, i32(cuda, *[s for s, _, _ in seqs]),
                      i32(cuda, *[n for _, n, _ in seqs]),
                      max(n for _, n, _ in seqs) if max_len is None else max_len, q_starts=starts,
                      max_q=max(counts) if max_q is None else max_q, accumulate=weights,
                      out=out[:, :c.QH * DIM], scratch=scratch)
    torch.cuda.synchronize()
    got, want, bound = host(out), np.full((rows, c.QH * DIM), 7.0), np.zeros((rows, c.QH * DIM))
    w_want, w_bound = before.copy(), np.zeros_like(before)
    at = 0
    for sid, n, m in seqs:
        o, b, s, sb = c.attend(q[at:at + m], sid, n)
        want[at:at + m], bound[at:at + m] = o, b
        blk, off = c.at(sid, n)
        w_want[blk, :, off] += s
        w_bound[blk, :, off] += sb
        at += m
    if stride:
        assert (got[:, c.QH * DIM:] == 7.0).all()
    d = np.abs(got[:, :c.QH * DIM] - want)
    assert (d <= bound).all(), f"out off by {np.max(d / np.maximum(bound, 1e-30))} bounds"
    w = host(cache.weights)
    if weights:
        d = np.abs(w - w_want)
        w_bound = w_bound + 2.0 ** -23 * (np.abs(w_want) + np.abs(before)) * (w_bound > 0)
        assert (d <= w_bound).all(), f"weights off by {np.max(d / np.maximum(w_bound, 1e-30))} bounds"
    else:
        np.testing.assert_array_equal(w, before)
    c.weights = w.astype(np.float32)
    return cache, table


# ----------------------------------------------------------- append and read
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("heads", [(32, 8), (5, 1), (3, 3)])
def test_append_equals_the_reference(cuda, dt, norm, heads):
    from dial_b200 import kv4

    c = Cache(3, 4, 80, *heads, dt=dt, fill=False, max_pos=500)
    cache, table = c.device(cuda)
    rows = 41
    sids = np.array([0] * 20 + [2] * 20 + [3], np.int32)
    slots = np.array(list(range(13, 33)) + list(range(20)) + [79], np.int32)
    slots[7] = -1  # a padding row
    pos = (slots + 300).astype(np.int32)
    x = act_round(c.rng.standard_normal((rows, (c.QH + 2 * c.H) * DIM)), dt)
    x[3] = 0
    x[4] *= 2.0 ** -13  # scales below e4m3's smallest
    x[5, ::7] *= 64
    x = act_round(x, dt)
    w = [act_round(1 + 0.2 * c.rng.standard_normal(DIM), dt) for _ in range(2)]
    ang = pos[:, None] * 1e6 ** (-np.arange(64) / 64)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda).to(dt)  # noqa: E731
    tab = np.arange(500)[:, None] * 1e6 ** (-np.arange(64) / 64)
    kw = dict(q_norm_w=t(w[0]), k_norm_w=t(w[1]), cos=t(np.cos(tab)), sin=t(np.sin(tab))) if norm else {}
    q = kv4.kv4_append(c.sh, cache, t(x), table, *(torch.from_numpy(a).to(cuda)
                                                   for a in (sids, slots, pos)), **kw)
    hd = x.reshape(rows, -1, DIM)
    cs = (act_round(np.cos(ang), dt), act_round(np.sin(ang), dt)) if norm else (None, None)
    eps = float(np.float32(1e-6))
    qr = norm_rope(hd[:, :c.QH], w[0] if norm else None, *cs, eps, dt)
    kr = norm_rope(hd[:, c.QH:c.QH + c.H], w[1] if norm else None, *cs, eps, dt)
    for m in range(rows):
        if slots[m] >= 0:
            c.put(sids[m], slots[m], kr[m], hd[m, c.QH + c.H:], pos[m])
            np.testing.assert_array_equal(host(q[m]), qr[m].reshape(-1))
    same_slabs(host(cache.pages), c.pages)
    np.testing.assert_array_equal(host(cache.weights), c.weights)
    np.testing.assert_array_equal(host(cache.positions), c.positions)
    # read back: the values themselves, and zeros past the length
    k, v = kv4.kv4_read(c.sh, cache, table, i32(cuda, 2, 0), i32(cuda, 20, 30), 27,
                        first=i32(cuda, 0, 5))
    for i, (sid, n, at) in enumerate(((2, 20, 0), (0, 30, 5))):
        kk, vv = c.values(sid, n)
        for got, want in ((k, kk), (v, vv)):
            want = act_round(want[at:at + 27], dt)
            np.testing.assert_array_equal(host(got[i])[:n - at], want)
            assert (host(got[i])[n - at:] == 0).all()


def test_append_of_nan_and_infinity(cuda):
    from dial_b200 import kv4

    c = Cache(5, 1, 16, 4, 2, fill=False)
    cache, table = c.device(cuda)
    x = act_round(c.rng.standard_normal((3, 8 * DIM)), BF16)
    x[0, 4 * DIM:5 * DIM:9] = np.nan
    x[0, 6 * DIM + 3] = np.inf
    x[1, 7 * DIM + 20] = -np.inf
    x[2, 4 * DIM:] = np.nan
    z = i32(cuda, 0, 0, 0)
    kv4.kv4_append(c.sh, cache, torch.from_numpy(x).to(cuda).to(BF16), table, z, i32(cuda, 0, 1, 2),
                   positions=z, want_q=False)
    for m in range(3):
        h = x[m].reshape(-1, DIM)
        c.put(0, m, h[4:6], h[6:], 0)
    same_slabs(host(cache.pages), c.pages)
    k, v = kv4.kv4_read(c.sh, cache, table, i32(cuda, 0), i32(cuda, 3), 3)
    assert np.isfinite(host(k)).all() and np.isfinite(host(v)).all()
    assert host(v)[0, 0, 0, 3] == 6 * 448 * c.v_scale and host(v)[0, 1, 1, 20] == -6 * 448 * c.v_scale
    assert (host(k)[0, 2] == 0).all() and (host(v)[0, 2] == 0).all()


def test_read_of_every_code_and_scale(cuda):
    from dial_b200 import kv4

    c = Cache(6, 1, 256 * 16, 2, 1, k_scale=1.0, v_scale=0.25, dt=F16)
    codes = np.tile(np.arange(16, dtype=np.uint8), 8)
    sc = np.array([s for s in range(127)], np.uint8)
    from kv4_case import pack
    for b in range(c.max_blocks):
        s = np.full((1, PAGE, 8), sc[b % 127], np.uint8)
        cc = np.broadcast_to(codes, (1, PAGE, DIM)).copy()
        c.pages[c.table[0, b]] = pack(cc, s, cc, s)
    cache, table = c.device(cuda)
    n = 256 * 16
    k, v = kv4.kv4_read(c.sh, cache, table, i32(cuda, 0), i32(cuda, n), n)
    kk, vv = c.values(0, n)
    np.testing.assert_array_equal(host(k)[0], act_round(kk, F16))
    np.testing.assert_array_equal(host(v)[0], act_round(vv, F16))


# ------------------------------------------------------------------ attention
HEADS = [(32, 8), (4, 4), (4, 2), (6, 2), (10, 2), (16, 2), (16, 1)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("dt", [BF16, F16])
def test_attention_single_tokens(cuda, heads, dt):
    c = Cache(11, 9, 700, *heads, dt=dt)
    lens = [1, 2, 15, 16, 17, 255, 256, 700, 0]
    check_attention(c, cuda, [(8 - i, n, 1) for i, n in enumerate(lens)])
    check_attention(c, cuda, [(3, 33, 1)], weights=False)


@pytest.mark.parametrize("heads", [(32, 8), (3, 3), (10, 2), (16, 1)])
@pytest.mark.parametrize("weights", [False, True])
def test_attention_few_queries(cuda, heads, weights):
    c = Cache(12, 8, 300, *heads, dt=F16 if heads[0] == 32 else BF16)
    check_attention(c, cuda, [(0, 300, 5), (1, 5, 5), (2, 3, 5), (4, 1, 1), (3, 17, 2), (6, 0, 3),
                              (5, 64, 0), (7, 129, 8)], weights=weights, spare_rows=3)


@pytest.mark.parametrize("queries,lens", [(16, (16, 40)), (33, (33, 90)), (64, (64, 257)),
                                          (129, (129, 400)), (200, (150, 200)), (20, (20, 2000)),
                                          (40, (700, 1300))])
@pytest.mark.parametrize("heads", [(8, 2), (5, 1), (2, 2)])
def test_attention_prompts(cuda, queries, lens, heads):
    c = Cache(13, 4, max(lens) + 16, *heads)
    check_attention(c, cuda, [(2, lens[1], queries), (0, lens[0], queries), (3, 7, 3)],
                    spare_rows=1, stride=64)


@pytest.mark.parametrize("weights", [False, True])
def test_attention_of_many_ragged_sequences(cuda, weights):
    """More sequences than one launch takes, most of them short or empty, a few
    long: ranges with many segments, and segments over many ranges."""
    c = Cache(19, 300, 900, 4, 2)
    lens = [int(n) for n in c.rng.integers(0, 40, 300)]
    for i, n in ((7, 900), (150, 777), (151, 0), (299, 899)):
        lens[i] = n
    check_attention(c, cuda, [(s, n, 1) for s, n in enumerate(lens)], weights=weights)


@pytest.mark.parametrize("weights", [False, True])
def test_ranges_of_many_ragged_sequences(cuda, weights):
    """The same with one sequence too long for a CTA a segment, in a call of more
    sequences than one launch takes."""
    c = Cache(21, 270, 1100, 3, 1)
    lens = [int(n) for n in c.rng.integers(0, 30, 270)]
    lens[130], lens[131], lens[264], lens[269] = 1100, 1025, 1090, 0
    check_attention(c, cuda, [(s, n, 1) for s, n in enumerate(lens)], weights=weights)


@pytest.mark.parametrize("queries", [8, 9, 12, 13])
def test_attention_around_the_few_queries_rule(cuda, queries):
    c = Cache(22, 2, 1500, 8, 2)
    check_attention(c, cuda, [(0, 1500, queries), (1, 1023, queries)])
    check_attention(c, cuda, [(0, 1024, queries), (1, 1000, 3)], weights=False)


def test_many_sequences_of_many_queries(cuda):
    """More sequences than one launch takes, each with rows for several tiles,
    one of one query, one of none."""
    c = Cache(20, 530, 70, 4, 2)
    seqs = [(s, int(n), 33) for s, n in enumerate(c.rng.integers(0, 70, 530))]
    seqs[5], seqs[511], seqs[513] = (5, 70, 1), (511, 66, 70), (513, 12, 0)
    check_attention(c, cuda, seqs, spare_rows=2)


def test_attention_long_split(cuda):
    """One session long enough for every split, at an odd length; the largest
    score in the first and in the last slot."""
    for seed in (14, 15):
        c = Cache(seed, 2, 20011, 8, 2, dt=F16)
        check_attention(c, cuda, [(1, 20011, 1)])
        check_attention(c, cuda, [(0, 9001, 1), (1, 3, 1)], max_len=20011)


def test_attention_of_dominant_and_equal_scores(cuda):
    """Queries large enough that one slot takes all the weight, and zero
    queries, where every slot has the same."""
    c = Cache(16, 2, 1000, 8, 2)
    check_attention(c, cuda, [(0, 1000, 1), (1, 517, 1)], q_scale=40.0)
    check_attention(c, cuda, [(0, 1000, 1), (1, 517, 1)], q_scale=0.0)
    check_attention(c, cuda, [(0, 1000, 70), (1, 517, 40)], q_scale=30.0)


@pytest.mark.parametrize("queries", [1, 5, 40])
def test_attention_ignores_what_lies_past_the_end(cuda, queries):
    """Slots past a sequence's end, in its last page and in the pages after it, hold
    bytes that would decode to NaN."""
    c = Cache(18, 3, 400, 8, 2)
    lens = [300, 41, 129]
    for s, n in enumerate(lens):
        for slot in range(n, c.max_blocks * PAGE):
            b, o = c.table[s, slot // PAGE], slot % PAGE
            for part, w in ((0, 64), (1024, 64), (2048, 8), (2176, 8)):
                c.pages[b, :, part + w * o:part + w * (o + 1)] = 0xFF
    check_attention(c, cuda, [(s, n, min(n, queries)) for s, n in enumerate(lens)])
    check_attention(c, cuda, [(s, n, min(n, queries)) for s, n in enumerate(lens)], weights=False,
                    max_len=400)


def test_attention_scale_of_the_shape(cuda):
    from dial_b200 import kv4

    c = Cache(17, 1, 64, 4, 2)
    sh = kv4.make_shape(4, 2, c.max_blocks, c.pages.shape[0], k_scale=c.k_scale, v_scale=c.v_scale,
                        softmax_scale=0.03)
    cache, table = c.device(cuda)
    q = act_round(c.rng.standard_normal((1, 4 * DIM)), BF16)
    got = kv4.kv4_attention(sh, cache, torch.from_numpy(q).to(cuda).to(BF16), table, i32(cuda, 0),
                            i32(cuda, 61), 64)
    o, b, _, _ = c.attend(q, 0, 61, float(np.float32(0.03)))
    assert (np.abs(host(got) - o) <= b).all()


# ------------------------------------------------------------------- eviction
@pytest.mark.parametrize("n,keep,recent", [(1, 1, 0), (17, 16, 3), (100, 1, 1), (100, 99, 99),
                                           (1023, 512, 64), (1025, 1000, 0), (5000, 1777, 300),
                                           (40, 60, 10), (33, 0, 0), (0, 5, 5)])
@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_equals_the_reference(cuda, n, keep, recent, out_of_place):
    from dial_b200 import kv4

    cap = max(n, keep, 16)
    c = Cache(21, 5, cap, 4, 2)
    for s in range(5):  # positions that rise along the slots, other in each head
        b, o = c.at(s, cap)
        for h in range(2):
            c.positions[b, h, o] = np.cumsum(c.rng.integers(1, 3, cap))
    seqs = [(3, n), (1, max(0, n - 5)), (4, n // 2)]
    dst = c.table.copy()
    if out_of_place:
        dst[:] = -1
        kb = -(-keep // PAGE) if keep else 0
        extra = 3 * kb
        c.pages = np.concatenate([c.pages, c.pages[:1].repeat(extra, 0)])
        c.weights = np.concatenate([c.weights, c.weights[:1].repeat(extra, 0)])
        c.positions = np.concatenate([c.positions, c.positions[:1].repeat(extra, 0)])
        first = c.sh.num_blocks
        for i, (s, _) in enumerate(seqs):
            dst[s, :kb] = np.arange(first + i * kb, first + (i + 1) * kb)[:c.max_blocks]
        c.sh.num_blocks = first + extra
    cache, table = c.device(cuda)
    lens = i32(cuda, *[m for _, m in seqs])
    new = kv4.kv4_evict(c.sh, cache, table, i32(cuda, *[s for s, _ in seqs]), lens, cap, keep, recent,
                        dst_table=torch.from_numpy(dst).to(cuda) if out_of_place else None,
                        lens_out=lens if not out_of_place else None)
    want = [c.evict(s, m, keep, recent, dst) for s, m in seqs]
    assert host(new).tolist() == want
    np.testing.assert_array_equal(host(cache.pages), c.pages)
    np.testing.assert_array_equal(host(cache.weights), c.weights)
    np.testing.assert_array_equal(host(cache.positions), c.positions)


@pytest.mark.parametrize("kind", ["equal", "ties", "special", "protected"])
def test_evict_of_ties_and_special_weights(cuda, kind):
    from dial_b200 import kv4

    c = Cache(22, 1, 3000, 2, 2)
    b, o = c.at(0, 3000)
    c.positions[b, :, o] = np.arange(3000)[:, None]
    if kind == "equal":
        c.weights[:] = 0.25
    elif kind == "ties":
        c.weights = np.round(c.weights).astype(np.float32)
    elif kind == "special":
        pick = c.rng.integers(0, 7, c.weights.shape)
        c.weights = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 1e-42],
                             np.float32)[pick]
    else:  # more entries protected than kept: positions all alike
        c.positions[:] = 5
    cache, table = c.device(cuda)
    new = kv4.kv4_evict(c.sh, cache, table, i32(cuda, 0), i32(cuda, 3000), 3000, 1300, 200)
    assert host(new).tolist() == [c.evict(0, 3000, 1300, 200)]
    np.testing.assert_array_equal(host(cache.pages), c.pages)
    np.testing.assert_array_equal(host(cache.weights), c.weights)
    np.testing.assert_array_equal(host(cache.positions), c.positions)


# ---------------------------------------------------------- a session's life
def test_a_run_of_steps_with_eviction(cuda):
    """Prompt, decode steps with running weights, eviction at the capacity, and
    decoding on in the freed slots, three sessions at once, each step against
    the reference."""
    from dial_b200 import kv4

    c = Cache(31, 3, 96, 8, 2, max_pos=400)
    cache, table = c.device(cuda)
    tab = np.arange(400)[:, None] * 1e6 ** (-np.arange(64) / 64)
    cos, sin = (act_round(f(tab), BF16) for f in (np.cos, np.sin))
    w = act_round(1 + 0.1 * c.rng.standard_normal(DIM), BF16)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda).to(BF16)  # noqa: E731
    kw = dict(q_norm_w=t(w), k_norm_w=t(w), cos=t(cos), sin=t(sin))
    lens, seen = np.array([0, 0, 0]), np.array([0, 0, 0])
    steps = [np.array([90, 40, 7])] + [np.array([1, 1, 1])] * 9
    for step, counts in enumerate(steps):
        sids, slots, pos = [], [], []
        for s in range(3):
            sids += [s] * counts[s]
            slots += range(lens[s], lens[s] + counts[s])
            pos += range(seen[s], seen[s] + counts[s])
        lens, seen = lens + counts, seen + counts
        rows = len(sids)
        x = act_round(c.rng.standard_normal((rows, 12 * DIM)), BF16)
        q = kv4.kv4_append(c.sh, cache, t(x), table, i32(cuda, *sids), i32(cuda, *slots),
                           i32(cuda, *pos), **kw)
        hd = x.reshape(rows, -1, DIM)
        eps = float(np.float32(1e-6))
        qr = norm_rope(hd[:, :8], w, cos[pos], sin[pos], eps, BF16)
        kr = norm_rope(hd[:, 8:10], w, cos[pos], sin[pos], eps, BF16)
        np.testing.assert_array_equal(host(q), qr.reshape(rows, -1))
        for m in range(rows):
            c.put(sids[m], slots[m], kr[m], hd[m, 10:], pos[m])
        same_slabs(host(cache.pages), c.pages)
        starts = i32(cuda, 0, *np.cumsum(counts).tolist())
        out = kv4.kv4_attention(c.sh, cache, q, table, i32(cuda, 0, 1, 2), i32(cuda, *lens.tolist()),
                                96, q_starts=starts, max_q=int(counts.max()), accumulate=True)
        at, before = 0, c.weights.astype(np.float64)
        for s in range(3):
            o, b, ws, wb = c.attend(qr.reshape(rows, -1)[at:at + counts[s]], s, lens[s])
            assert (np.abs(host(out[at:at + counts[s]]) - o) <= b).all()
            blk, off = c.at(s, lens[s])
            got = host(cache.weights)[blk, :, off]
            assert (np.abs(got - before[blk, :, off] - ws) <= wb + 2.0 ** -22 * (got + 1e-30)).all()
            at += counts[s]
        c.weights = host(cache.weights).astype(np.float32)
        if step in (3, 6):
            full = [s for s in range(3) if lens[s] > 60]
            new = kv4.kv4_evict(c.sh, cache, table, i32(cuda, *full),
                                i32(cuda, *lens[full].tolist()), 96, 60, 20)
            for i, s in enumerate(full):
                assert int(new[i]) == c.evict(s, int(lens[s]), 60, 20)
                lens[s] = 60
            same_slabs(host(cache.pages), c.pages)
            np.testing.assert_array_equal(host(cache.weights), c.weights)
            np.testing.assert_array_equal(host(cache.positions), c.positions)


# ------------------------------------------- streams, graphs, devices, refusals
STATUS_BAD_ARGS = 0x104  # kStatusBadArgs (csrc/common.cuh)


def test_a_captured_step_replays_on_new_inputs(cuda):
    """append -> attention with weights -> eviction captured once and replayed with
    other rows, lengths and pages: as the same calls made eagerly."""
    from dial_b200 import kv4

    c = Cache(41, 3, 1024, 8, 2)
    base, table = c.device(cuda)
    runs = []
    for graph in (False, True):
        cache = kv4.Kv4Cache(base.pages.clone(), base.weights.clone(), base.positions.clone())
        x = torch.zeros(3, 12 * DIM, dtype=BF16, device=cuda)
        sids, slots, lens = i32(cuda, 0, 1, 2), i32(cuda, 0, 0, 0), i32(cuda, 0, 0, 0)
        pos = i32(cuda, 0, 0, 0)
        new = torch.zeros_like(lens)
        q = torch.zeros(3, 8 * DIM, dtype=BF16, device=cuda)
        out = torch.zeros_like(q)
        s1 = torch.empty(kv4.attention_scratch_bytes(c.sh, 3, 3, 1, 1024, True) + 16, dtype=torch.uint8,
                         device=cuda)
        s2 = torch.empty(kv4.evict_scratch_bytes(c.sh, 3, 1024, 700), dtype=torch.uint8, device=cuda)

        def step():
            kv4.kv4_append(c.sh, cache, x, table, sids, slots, pos, q_out=q)
            kv4.kv4_attention(c.sh, cache, q, table, sids, lens, 1024, accumulate=True, out=out,
                              scratch=s1)
            kv4.kv4_evict(c.sh, cache, table, sids, lens, 1024, 700, 100, lens_out=new, scratch=s2)

        if graph:
            side = torch.cuda.Stream(cuda)
            side.wait_stream(torch.cuda.current_stream(cuda))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
                step()
            torch.cuda.synchronize()
        got = []
        gen = torch.Generator(device=cuda)
        gen.manual_seed(1)
        for n in ([900, 1, 33], [701, 700, 2], [17, 1000, 699]):
            x.copy_(torch.randn(x.shape, generator=gen, device=cuda))
            lens.copy_(i32(cuda, *n))
            slots.copy_(lens - 1)
            pos.copy_(lens + 3)
            g.replay() if graph else step()
            got.append([t.clone() for t in (out, new, cache.pages, cache.weights, cache.positions)])
        torch.cuda.synchronize()
        runs.append(got)
    for eager, replayed in zip(*runs):
        for a, b in zip(eager, replayed):
            assert torch.equal(a, b)


def test_two_streams_with_scratch_of_their_own(cuda):
    """Calls that overlap in time, each with its own scratch, on streams other than
    their tensors', as the same calls alone."""
    from dial_b200 import kv4

    c = Cache(42, 2, 3000, 8, 2)
    cache, table = c.device(cuda)
    q = (torch.randn(2, 8 * DIM, device=cuda) * 2).to(BF16)
    qs = (torch.randn(300, 8 * DIM, device=cuda) * 2).to(BF16)

    def call(kind):
        if kind == 0:
            return kv4.kv4_attention(c.sh, cache, q, table, i32(cuda, 0, 1), i32(cuda, 3000, 2999), 3000)
        return kv4.kv4_attention(c.sh, cache, qs, table, i32(cuda, 1), i32(cuda, 2500), 3000,
                                 q_starts=i32(cuda, 0, 300), max_q=300)

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    for _ in range(10):
        got = [None, None]
        for k, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream(cuda))
            with torch.cuda.stream(s):
                got[k] = call(k)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_repeated_calls_give_the_same_bits(cuda):
    c = Cache(43, 4, 5000, 32, 8)
    cache, table = c.device(cuda)
    q = (torch.randn(4, 32 * DIM, device=cuda) * 2).to(BF16)
    lens = i32(cuda, 5000, 17, 4001, 900)
    from dial_b200 import kv4

    outs, weights = [], []
    for _ in range(6):
        w = kv4.Kv4Cache(cache.pages, cache.weights.clone(), cache.positions)
        outs.append(kv4.kv4_attention(c.sh, w, q, table, i32(cuda, 0, 1, 2, 3), lens, 5000, accumulate=True))
        weights.append(w.weights)
    assert all(torch.equal(o, outs[0]) for o in outs) and all(torch.equal(w, weights[0]) for w in weights)


def test_pages_past_four_gigabytes(cuda):
    """Pages whose byte offset passes 32 bits, at the end of a pool of 5 GB."""
    from dial_b200 import kv4

    c = Cache(44, 1, 200, 8, 4)
    blocks = (5 << 30) // (4 * 2304)
    small, _ = c.device(cuda)
    big = kv4.Kv4Cache(torch.empty(blocks, 4, 2304, dtype=torch.uint8, device=cuda),
                       torch.zeros(blocks, 4, PAGE, device=cuda),
                       torch.zeros(blocks, 4, PAGE, dtype=torch.int32, device=cuda))
    shift = blocks - c.pages.shape[0]
    big.pages[shift:] = small.pages
    big.weights[shift:] = small.weights
    c.table = c.table + shift
    c.sh.num_blocks = blocks
    table = torch.from_numpy(c.table).to(cuda)
    q = (torch.randn(1, 8 * DIM, device=cuda) * 2).to(BF16)
    out = kv4.kv4_attention(c.sh, big, q, table, i32(cuda, 0), i32(cuda, 200), 200, accumulate=True)
    new = kv4.kv4_evict(c.sh, big, table, i32(cuda, 0), i32(cuda, 200), 200, 90)
    k, v = kv4.kv4_read(c.sh, big, table, i32(cuda, 0), new, 90)
    c.table = c.table - shift
    o, b, s, _ = c.attend(host(q), 0, 200)
    assert (np.abs(host(out) - o) <= b).all()
    # the same on the small pool, bit for bit
    ref, table = c.device(cuda)
    c.sh.num_blocks = c.pages.shape[0]
    out2 = kv4.kv4_attention(c.sh, ref, q, table, i32(cuda, 0), i32(cuda, 200), 200, accumulate=True)
    kv4.kv4_evict(c.sh, ref, table, i32(cuda, 0), i32(cuda, 200), 200, 90)
    k2, v2 = kv4.kv4_read(c.sh, ref, table, i32(cuda, 0), new, 90)
    assert int(new[0]) == 90 and torch.equal(out, out2) and torch.equal(k, k2) and torch.equal(v, v2)
    assert torch.equal(big.weights[shift:], ref.weights) and torch.equal(big.pages[shift:], ref.pages)
    del big
    torch.cuda.empty_cache()


def test_bad_rows_are_left_out_and_reported(cuda):
    """Sessions, slots, positions, lengths and block ids out of range: the status is
    set, the good rows are as without the bad ones, memory outside is untouched."""
    import dial_b200
    from dial_b200 import kv4

    c = Cache(45, 4, 160, 8, 2, max_pos=200)
    good, table = c.device(cuda)
    x = torch.randn(6, 12 * DIM, device=cuda).to(BF16)
    ang = torch.zeros(200, 64, dtype=BF16, device=cuda)
    # rows 1-4 are bad: session 4, slot past the table, position past the tables, negative session
    cache = kv4.Kv4Cache(good.pages.clone(), good.weights.clone(), good.positions.clone())
    q = kv4.kv4_append(c.sh, cache, x, table, i32(cuda, 0, 4, 1, 1, -1, 2), i32(cuda, 5, 1, 160, 7, 3, 9),
                       i32(cuda, 1, 1, 1, 200, 1, 1), cos=ang + 1, sin=ang,
                       q_out=torch.full((6, 8 * DIM), 3.0, dtype=BF16, device=cuda))
    assert dial_b200.device_status(clear=True) == STATUS_BAD_ARGS
    assert (q[1:5] == 3.0).all() and (q[0] != 3.0).any() and (q[5] != 3.0).any()
    want = kv4.Kv4Cache(good.pages.clone(), good.weights.clone(), good.positions.clone())
    kv4.kv4_append(c.sh, want, x[[0, 5]].contiguous(), table, i32(cuda, 0, 2), i32(cuda, 5, 9), i32(cuda, 1, 1),
                   cos=ang + 1, sin=ang)
    for a, b in ((cache.pages, want.pages), (cache.weights, want.weights), (cache.positions, want.positions)):
        assert torch.equal(a, b)
    assert dial_b200.device_status() == 0
    # attention: a bad session, a length past max_len, a negative one, rows out of order
    for queries in (1, 40):
        starts = i32(cuda, *[i * queries for i in range(5)])
        qq = (torch.randn(4 * queries, 8 * DIM, device=cuda)).to(BF16)
        for bad_sids, bad_lens in (((0, 9, 2, 3), (150, 9, 80, 0)), ((0, 1, 2, 3), (150, 161, 80, -1))):
            w = good.weights.clone()
            cc = kv4.Kv4Cache(good.pages, w, good.positions)
            out = torch.full_like(qq, 5.0)
            kv4.kv4_attention(c.sh, cc, qq, table, i32(cuda, *bad_sids), i32(cuda, *bad_lens), 160,
                              q_starts=starts, max_q=queries, accumulate=True, out=out)
            assert dial_b200.device_status(clear=True) == STATUS_BAD_ARGS
            for i in (0, 2):
                o, b, _, _ = c.attend(host(qq[i * queries:(i + 1) * queries]), i, (150, 0, 80)[i])
                d = np.abs(host(out[i * queries:(i + 1) * queries]) - o)
                assert (d <= b).all()
            assert (out[queries:2 * queries] == 5.0).all()
            w_sum = host(w - good.weights)
            blk, _ = c.at(1, 160)
            assert (w_sum[blk] == 0).all()
    # block ids outside the pool: page 0 is read, nothing is written outside
    bad = table.clone()
    bad[0, 2] = c.sh.num_blocks
    bad[1, 0] = -7
    out = kv4.kv4_attention(c.sh, good, x[:2, :8 * DIM], bad, i32(cuda, 0, 1), i32(cuda, 100, 30), 160)
    assert dial_b200.device_status(clear=True) == STATUS_BAD_ARGS
    c2 = Cache(45, 4, 160, 8, 2, max_pos=200)
    c2.pages, c2.table = c.pages, c.table.copy()
    c2.table[0, 2] = c2.table[1, 0] = 0
    for i, n in ((0, 100), (1, 30)):
        o, b, _, _ = c2.attend(host(x[i:i + 1, :8 * DIM]), i, n)
        assert (np.abs(host(out[i:i + 1]) - o) <= b).all()
    before = good.pages.clone()
    kv4.kv4_append(c.sh, good, x[:1], bad, i32(cuda, 1), i32(cuda, 3), i32(cuda, 0))
    assert torch.equal(good.pages, before)
    assert dial_b200.device_status(clear=True) == STATUS_BAD_ARGS
    # eviction of a bad sequence: its length stays, the good one's is cut
    lens = i32(cuda, 150, 170, 80)
    kv4.kv4_evict(c.sh, good, table, i32(cuda, 0, 1, 2), lens, 160, 50, 10, lens_out=lens)
    assert lens.tolist() == [50, 170, 50]
    assert dial_b200.device_status(clear=True) == STATUS_BAD_ARGS


def test_append_and_read_of_strided_rows(cuda):
    """qkv, q_out, q and out as columns of wider tensors; the columns beside stay."""
    from dial_b200 import kv4

    c = Cache(46, 1, 64, 4, 2)
    cache, table = c.device(cuda)
    wide = torch.randn(5, 8 * DIM + 64, device=cuda).to(BF16)
    qw = torch.full((5, 4 * DIM + 128), 9.0, dtype=BF16, device=cuda)
    kv4.kv4_append(c.sh, cache, wide[:, 64:], table, i32(cuda, 0, 0, 0, 0, 0), i32(cuda, 0, 1, 2, 3, 4),
                   i32(cuda, 0, 1, 2, 3, 4), q_out=qw[:, 128:])
    assert (qw[:, :128] == 9.0).all() and torch.equal(qw[:, 128:], wide[:, 64:64 + 4 * DIM])
    ref, _ = c.device(cuda)
    kv4.kv4_append(c.sh, ref, wide[:, 64:].contiguous(), table, i32(cuda, 0, 0, 0, 0, 0),
                   i32(cuda, 0, 1, 2, 3, 4), i32(cuda, 0, 1, 2, 3, 4))
    assert torch.equal(cache.pages, ref.pages)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_prompt_rows_on_sixteen_byte_boundaries(cuda, dt):
    """q and out that start on 16-byte but not on 32-byte boundaries, whole items and
    items cut over the GPU: the bits of an aligned call, the columns beside untouched."""
    from dial_b200 import kv4

    c = Cache(48, 2, 2600, 8, 2, dt=dt)
    cache, table = c.device(cuda)
    width, rows = 8 * DIM, 230
    wide = (torch.randn(rows, width + 24, device=cuda) * 2).to(dt)
    out = torch.full((rows, width + 24), 3.0, dtype=dt, device=cuda)
    args = (table, i32(cuda, 1, 0), i32(cuda, 2600, 70), 2600, i32(cuda, 0, 200, 230), 200)
    kv4.kv4_attention(c.sh, cache, wide[:, 8:8 + width], *args, out=out[:, 8:8 + width])
    want = kv4.kv4_attention(c.sh, cache, wide[:, 8:8 + width].contiguous(), *args)
    assert torch.equal(out[:, 8:8 + width], want)
    assert (out[:, :8] == 3.0).all() and (out[:, 8 + width:] == 3.0).all()
    o, b, _, _ = c.attend(host(wide[:200, 8:8 + width]), 1, 2600)
    assert (np.abs(host(want[:200]) - o) <= b).all()


def test_evict_twice_and_the_same_bits(cuda):
    """An eviction repeated on what it left changes nothing; two runs give the same
    bits; sessions evicted beside each other as one by one."""
    from dial_b200 import kv4

    c = Cache(49, 3, 900, 4, 2)
    runs = []
    for one_by_one in (False, True, False):
        cache, table = c.device(cuda)
        if one_by_one:
            new = torch.cat([kv4.kv4_evict(c.sh, cache, table, i32(cuda, s), i32(cuda, n), 900, 300, 40)
                             for s, n in ((0, 900), (1, 299), (2, 640))])
        else:
            new = kv4.kv4_evict(c.sh, cache, table, i32(cuda, 0, 1, 2), i32(cuda, 900, 299, 640), 900, 300, 40)
        runs.append((new, cache.pages.clone(), cache.weights.clone(), cache.positions.clone()))
        again = kv4.kv4_evict(c.sh, cache, table, i32(cuda, 0, 1, 2), new, 900, 300, 40)
        assert again.tolist() == [300, 299, 300]
        assert torch.equal(cache.pages, runs[-1][1]) and torch.equal(cache.weights, runs[-1][2])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_sequences_without_queries(cuda):
    """max_q 0, and sequences whose rows are all spare."""
    c = Cache(50, 2, 60, 8, 2)
    check_attention(c, cuda, [(0, 40, 0), (1, 0, 0)], spare_rows=3)
    check_attention(c, cuda, [(0, 40, 0), (1, 33, 0)], spare_rows=3, max_q=5, weights=False)


def test_empty_calls(cuda):
    from dial_b200 import kv4

    c = Cache(47, 1, 64, 4, 2)
    cache, table = c.device(cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    q = torch.zeros(0, 4 * DIM, dtype=BF16, device=cuda)
    assert kv4.kv4_attention(c.sh, cache, q, table, none, none, 64).shape == (0, 4 * DIM)
    k, _ = kv4.kv4_read(c.sh, cache, table, none, none, 3)
    assert k.shape == (0, 3, 2, DIM)
    assert kv4.kv4_append(c.sh, cache, torch.zeros(0, 8 * DIM, dtype=BF16, device=cuda), table, none, none,
                          none).shape == (0, 4 * DIM)
    assert kv4.kv4_evict(c.sh, cache, table, none, none, 64, 8).shape == (0,)
    # max_len 0: every query sees nothing
    out = kv4.kv4_attention(c.sh, cache, torch.ones(2, 4 * DIM, dtype=BF16, device=cuda), table,
                            i32(cuda, 0, 0), i32(cuda, 0, 0), 0)
    assert (out == 0).all()
    out = kv4.kv4_attention(c.sh, cache, torch.ones(90, 4 * DIM, dtype=BF16, device=cuda), table, i32(cuda, 0),
                            i32(cuda, 0), 0, q_starts=i32(cuda, 0, 90), max_q=90, accumulate=True)
    assert (out == 0).all()
    torch.cuda.synchronize()
