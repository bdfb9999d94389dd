"""Cases of the 4-bit KV cache operators: what a session's serving loop does
with a cache of e2m1 codes (two a byte, an e4m3 scale for every 16 dims) in
16-token pages.

  append     rows of q | k | v: q/k RMSNorm and RoPE, k and v quantised into
             their slots; the rotated q and the values now cached come back
             (the values through the read operator).
  attention  queries over the cached slots of their sessions, one token a
             session or many, optionally adding each slot's softmax weight to
             its running sum.
  evict      the slots of each session and kv head cut to `keep` by that sum,
             the newest `recent` protected, into pages of their own; the kept
             entries come back through the read operator.

Every case states its sizes as plain values; ragged lengths follow from the
case alone, so that its work does, and the contents from the seed.
"""

import math
import random
import sys

import numpy as np
import torch

own = False

PAGE = 16            # tokens in a page
DIM = 128            # head dim
GROUP = 16           # dims that share a scale
SLAB = 2304          # bytes of one page of one kv head
EPS = 1e-6
THETA = 1e6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ----------------------------------------------------------------- cases
def _append(name, rows, seqs, q_heads, kv_heads, dtype, start, norm=True):
    return {"name": name, "op": "append", "rows": rows, "seqs": seqs, "q_heads": q_heads,
            "kv_heads": kv_heads, "dtype": dtype, "start": start, "norm": norm}


def _attention(name, seqs, shortest, longest, queries, q_heads, kv_heads, dtype, weights):
    return {"name": name, "op": "attention", "seqs": seqs, "shortest": shortest,
            "longest": longest, "queries": queries, "q_heads": q_heads, "kv_heads": kv_heads,
            "dtype": dtype, "weights": weights}


def _evict(name, seqs, shortest, longest, keep, recent, q_heads, kv_heads, dtype):
    return {"name": name, "op": "evict", "seqs": seqs, "shortest": shortest, "longest": longest,
            "keep": keep, "recent": recent, "q_heads": q_heads, "kv_heads": kv_heads,
            "dtype": dtype}


def listed():
    return [
        # one decoded token of one session, in the 8B decoder's heads
        _append("append_token", 1, 1, 32, 8, "bf16", 200),
        # the ragged decode step of many sessions of the 27B-class decoder's
        # heads; rows already normed and rotated by the caller
        _append("append_step_f16", 37, 37, 40, 8, "f16", 1500, norm=False),
        # a 2048-token prompt
        _append("append_prompt", 2048, 1, 32, 8, "bf16", 0),
        # one session shortly after its 128-token prompt: latency alone
        _attention("decode_short", 1, 201, 201, 1, 32, 8, "bf16", False),
        # 32 ragged sessions of 128 to 8192 cached tokens
        _attention("decode_ragged", 32, 128, 8192, 1, 32, 8, "bf16", False),
        # one very long session: few rows, the cache split over the whole GPU
        _attention("decode_long", 1, 131071, 131071, 1, 40, 8, "f16", False),
        # a ragged step that keeps the running weights for a later eviction
        _attention("decode_weights", 9, 900, 30001, 1, 32, 8, "bf16", True),
        # five drafted tokens a session, verified together
        _attention("verify_five", 8, 700, 4099, 5, 32, 8, "f16", True),
        # a 2048-token prompt attending to itself
        _attention("prompt", 1, 2048, 2048, 2048, 32, 8, "bf16", False),
        # a chunk of a long prompt over what is cached already, with weights
        _attention("chunk_weights", 2, 9500, 16897, 512, 40, 8, "bf16", True),
        # one session that has just passed its budget
        _evict("evict_session", 1, 1100, 1100, 1024, 128, 32, 8, "bf16"),
        # many sessions halved at once
        _evict("evict_many", 16, 3500, 8192, 4096, 512, 32, 8, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    q_heads, kv_heads = rng.choice([(32, 8), (40, 8), (16, 8), (8, 8), (16, 4), (32, 4), (6, 2)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    op = rng.choice(["append", "attention", "attention", "attention", "evict"])
    if op == "append":
        rows = _log(rng, 1, 2048)
        seqs = min(rows, rng.choice([1, 1, 2, 7, rows]))
        c = _append("", rows, seqs, q_heads, kv_heads, dtype, rng.randrange(0, 2000),
                    rng.random() < 0.7)
    elif op == "attention":
        seqs = _log(rng, 1, 48)
        kind = rng.choice(["token", "token", "few", "many"])
        if kind == "many":
            seqs = min(seqs, 4)
            queries = _log(rng, 33, 1024)
            longest = queries + _log(rng, 1, min(16000 * 512 // queries, 120000) // seqs)
        else:
            queries = 1 if kind == "token" else rng.randrange(2, 25)
            longest = queries + _log(rng, 1, 120000 // (seqs * (1 if kind == "token" else 2)))
        shortest = rng.randrange(min(queries, longest), longest + 1)
        c = _attention("", seqs, shortest, longest, queries, q_heads, kv_heads, dtype,
                       rng.random() < 0.5)
    else:
        seqs = _log(rng, 1, 16)
        longest = _log(rng, 40, 8192)
        shortest = rng.randrange(max(1, longest // 3), longest + 1)
        keep = rng.randrange(max(1, longest // 4), longest)
        c = _evict("", seqs, shortest, longest, keep, rng.randrange(0, keep + 1), q_heads,
                   kv_heads, dtype)
    del c["name"]
    return c


def _lengths(case):
    """Cached slots of each session: spread over the case's range by the case
    alone, the longest there."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    r = random.Random(7919 * n + 31 * lo + hi)
    got = [r.randint(lo, hi) for _ in range(n)]
    got[r.randrange(n)] = hi
    return got


def _queries(case, lens):
    """Query tokens of each session: all of `queries` for the first, fewer for
    some of the others, never more than there are slots."""
    q = case["queries"]
    r = random.Random(104729 * q + len(lens))
    return [min(n, q if i == 0 or r.random() < 0.5 else r.randint((q + 1) // 2, q))
            for i, n in enumerate(lens)]


def _row_counts(case):
    """Rows of each session of an append, as even as they go."""
    base, more = divmod(case["rows"], case["seqs"])
    return [base + (i < more) for i in range(case["seqs"])]


# --------------------------------------------------------------- the format
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _encode(x, g):
    """x [..., 128] float32 to (codes uint8 [..., 64], e4m3 scales [..., 8])."""
    x = torch.nan_to_num(x, nan=0.0)
    grp = x.reshape(*x.shape[:-1], DIM // GROUP, GROUP)
    amax = grp.abs().amax(dim=-1)
    scale = (amax / 6.0 / g).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float().unsqueeze(-1) * g
    a = torch.where(s > 0, grp.abs() / s, torch.zeros_like(grp))
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5.0))
    code = code | (torch.signbit(grp) & (s > 0)).to(torch.uint8) << 3
    code = code.reshape(*x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def _decode(codes, scales, g):
    """The values of codes [..., 64] and e4m3 scales [..., 8], float32."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*codes.shape[:-1], DIM)
    v = lut[both.int()].reshape(*codes.shape[:-1], DIM // GROUP, GROUP)
    return (v * (scales.float() * g).unsqueeze(-1)).reshape(*codes.shape[:-1], DIM)


def _slab(kc, ks, vc, vs):
    """Pages [..., 16, .] of k and v codes and scales as slabs [..., 2304]."""
    flat = lambda t: t.contiguous().view(torch.uint8).reshape(*t.shape[:-2], -1)  # noqa: E731
    return torch.cat([flat(kc), flat(vc), flat(ks), flat(vs)], dim=-1)


def _unslab(slab):
    """Slabs [..., 2304] as (k codes, k scales, v codes, v scales) of 16 tokens."""
    part = lambda a, b, w: slab[..., a:b].contiguous().reshape(*slab.shape[:-1], PAGE, w)  # noqa: E731
    e4m3 = torch.float8_e4m3fn
    return (part(0, 1024, 64), part(2048, 2176, 8).view(e4m3),
            part(1024, 2048, 64), part(2176, 2304, 8).view(e4m3))


# ------------------------------------------------------------------ inputs
def _random_pages(gen, dev, blocks, kv_heads, k_scale, v_scale):
    """Pages whose keys have a few strong channels, as rotated keys do."""
    out = torch.empty(blocks, kv_heads, SLAB, dtype=torch.uint8, device=dev)
    chan = torch.exp(0.5 * torch.randn(kv_heads, 1, DIM, generator=gen, device=dev))
    step = max(1, (1 << 24) // (kv_heads * PAGE * DIM))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        k = torch.randn(n, kv_heads, PAGE, DIM, generator=gen, device=dev) * chan
        v = torch.randn(n, kv_heads, PAGE, DIM, generator=gen, device=dev) * 0.5
        out[at:at + n] = _slab(*_encode(k, k_scale), *_encode(v, v_scale))
    return out


def _table(gen, dev, sessions, max_blocks, spare):
    """A block table of pages in no order, and how many pages the pool has."""
    total = sessions * max_blocks + spare
    perm = torch.randperm(total, generator=gen, device=dev).int()
    return perm[:sessions * max_blocks].reshape(sessions, max_blocks).contiguous(), total


def _rope_tables(dev, dtype, rows):
    inv = 1.0 / THETA ** (torch.arange(0, DIM, 2, device=dev, dtype=torch.float64) / DIM)
    ang = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * inv
    return ang.cos().to(dtype), ang.sin().to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    op, dt, kvh, qh = case["op"], TYPES[case["dtype"]], case["kv_heads"], case["q_heads"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    st = {"case": dict(case), "k_scale": 0.5, "v_scale": 0.0625, "keep_by": {}}
    if op == "append":
        counts = _row_counts(case)
        last = case["start"] + max(counts)
        max_blocks = -(-last // PAGE) + 1
        st["table"], blocks = _table(gen, dev, case["seqs"] + 1, max_blocks, 3)
        st["pages"] = _random_pages(gen, dev, blocks, kvh, st["k_scale"], st["v_scale"])
        sids, slots = [], []
        for s, n in enumerate(counts):
            sids += [s] * n
            slots += range(case["start"], case["start"] + n)
        st["sids"], st["slots"] = i32(sids), i32(slots)
        # evicted sessions hold fewer slots than tokens seen
        st["at"] = st["slots"] + 11
        st["qkv"] = torch.randn(case["rows"], (qh + 2 * kvh) * DIM, generator=gen, device=dev).to(dt)
        st["max_pos"] = last + 16
        if case["norm"]:
            w = lambda: (1 + 0.2 * torch.randn(DIM, generator=gen, device=dev)).to(dt)  # noqa: E731
            st["q_norm"], st["k_norm"] = w(), w()
            st["cos"], st["sin"] = _rope_tables(dev, dt, st["max_pos"])
        st["ends"] = st["slots"] + 1
    else:
        lens = _lengths(case)
        st["max_len"] = max(lens)
        max_blocks = -(-max(lens) // PAGE)
        n = case["seqs"]
        st["sids"] = torch.randperm(n + 1, generator=gen, device=dev)[:n].int()
        st["lens"] = i32(lens)
        if op == "attention":
            st["table"], blocks = _table(gen, dev, n + 1, max_blocks, 1)
            qs = _queries(case, lens)
            st["max_q"] = max(qs)
            st["starts"] = i32([0] + np.cumsum(qs).tolist())
            st["q"] = (1.5 * torch.randn(sum(qs), qh * DIM, generator=gen, device=dev)).to(dt)
        else:
            keep_blocks = -(-case["keep"] // PAGE)
            both, blocks = _table(gen, dev, n + 1, max_blocks + keep_blocks, 1)
            st["table"] = both[:, :max_blocks].contiguous()
            st["dst_table"] = torch.cat([both[:, max_blocks:], torch.full_like(
                both[:, :max_blocks - keep_blocks], -1)], dim=1).contiguous()
        st["pages"] = _random_pages(gen, dev, blocks, kvh, st["k_scale"], st["v_scale"])
        # running weights as some steps of attention leave them: a few heavy
        # slots, a long tail, a sum of a few steps' worth
        st["weights"] = torch.exp(2.0 * torch.randn(blocks, kvh, PAGE, generator=gen, device=dev))
        st["weights"] *= 0.5 / st["max_len"]
        # positions rise along a session's slots, not one by one
        pos = torch.empty(blocks, kvh, PAGE, dtype=torch.int32, device=dev)
        rise = torch.randint(1, 3, (n + 1, max_blocks * PAGE), generator=gen, device=dev).cumsum(1)
        pos[:] = torch.randint(0, 1 << 20, pos.shape, generator=gen, device=dev).int()
        pos[st["table"].long()] = rise.int().reshape(n + 1, max_blocks, 1, PAGE).expand(
            -1, -1, kvh, -1)
        st["positions"] = pos
    return st


# ------------------------------------------------------- the plain operators
def _put(st, sids, slots, k, v):
    """Rows of k and v, float32 [rows, kv_heads, 128], into their slots."""
    block = st["table"][sids.long(), (slots // PAGE).long()].long()
    off = (slots % PAGE).long()
    heads = torch.arange(k.shape[1], device=k.device)[None, :, None]
    byte = torch.arange(64, device=k.device)
    for x, g, codes_at, scales_at in ((k, st["k_scale"], 0, 2048), (v, st["v_scale"], 1024, 2176)):
        codes, scales = _encode(x, g)
        at = codes_at + 64 * off[:, None, None] + byte
        st["pages"][block[:, None, None], heads, at] = codes
        at = scales_at + 8 * off[:, None, None] + byte[:8]
        st["pages"][block[:, None, None], heads, at] = scales.view(torch.uint8)


def _get(st, table, sids, first, lens, count, dtype):
    """The values of `count` slots of each session from `first`, zeros from
    its `lens` on: k and v [sessions, count, kv_heads, 128]."""
    slot = first.long()[:, None] + torch.arange(count, device=sids.device)
    fine = slot < lens.long()[:, None]
    slot = torch.where(fine, slot, torch.zeros_like(slot))
    block = table[sids.long()].gather(1, slot // PAGE).long()
    block = torch.where(fine, block, torch.zeros_like(block))
    kc, ks, vc, vs = _unslab(st["pages"])
    got = []
    for codes, scales, g in ((kc, ks, st["k_scale"]), (vc, vs, st["v_scale"])):
        c = codes.permute(0, 2, 1, 3)[block, slot % PAGE]
        s = scales.view(torch.uint8).permute(0, 2, 1, 3)[block, slot % PAGE]
        x = _decode(c, s.view(torch.float8_e4m3fn), g)
        got.append(torch.where(fine[:, :, None, None], x, torch.zeros_like(x)).to(dtype))
    return got


def _norm_rope(x, w, cos, sin, dtype):
    """Rows [rows, heads, 128] of `dtype`: RMSNorm and RoPE, each step rounded
    to `dtype`; sums in 64 bits, since a step's result may lie next to a border."""
    r = lambda t: t.to(dtype).float()  # noqa: E731
    ss = x.double().square().sum(dim=-1, keepdim=True)
    y = r(r(x.float() / r((ss / DIM + EPS).sqrt())) * w.float())
    a, b = y[..., :DIM // 2], y[..., DIM // 2:]
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat([r(r(a * c) - r(b * s)), r(r(a * s) + r(b * c))], dim=-1)


def _plain_append(st):
    case = st["case"]
    dt, qh, kvh = TYPES[case["dtype"]], case["q_heads"], case["kv_heads"]
    x = st["qkv"].reshape(case["rows"], qh + 2 * kvh, DIM)
    q, k, v = x[:, :qh], x[:, qh:qh + kvh].float(), x[:, qh + kvh:].float()
    if case["norm"]:
        cos, sin = st["cos"][st["at"].long()], st["sin"][st["at"].long()]
        q = _norm_rope(q, st["q_norm"], cos, sin, dt)
        k = _norm_rope(k, st["k_norm"], cos, sin, dt)
    _put(st, st["sids"], st["slots"], k, v)
    k, v = _get(st, st["table"], st["sids"], st["slots"], st["ends"], 1, dt)
    return {"q": q.reshape(case["rows"], -1).to(dt), "k": k, "v": v}


def _plain_attention(st):
    case = st["case"]
    dt, qh, kvh, n = TYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["seqs"]
    rep, most, L = qh // kvh, st["max_q"], st["max_len"]
    dev = st["q"].device
    blocks = -(-L // PAGE)
    kc, ks, vc, vs = _unslab(st["pages"][st["table"][st["sids"].long(), :blocks].long()])
    seq = lambda t: t.transpose(2, 3).reshape(n, blocks * PAGE, kvh, DIM)[:, :L].transpose(1, 2)  # noqa: E731
    k, v = seq(_decode(kc, ks, st["k_scale"])), seq(_decode(vc, vs, st["v_scale"]))
    starts = st["starts"].long()
    counts = starts[1:] - starts[:-1]
    tok = torch.arange(most, device=dev)
    there = tok < counts[:, None]
    row = torch.where(there, starts[:-1, None] + tok, torch.zeros_like(tok))
    q = st["q"][row].float().reshape(n, most, kvh, rep, DIM).permute(0, 2, 1, 3, 4)
    s = (q.reshape(n, kvh, most * rep, DIM) @ k.transpose(2, 3)) / math.sqrt(DIM)
    seen = st["lens"].long()[:, None] - counts[:, None] + 1 + tok      # slots a query sees
    seen = torch.where(there, seen, torch.zeros_like(seen))
    mask = torch.arange(L, device=dev) < seen[:, :, None]
    mask = mask[:, None, :, None].expand(n, 1, most, rep, L).reshape(n, 1, most * rep, L)
    s = s.masked_fill(~mask, -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    del s, mask
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = (p @ v).reshape(n, kvh, most, rep, DIM).permute(0, 2, 1, 3, 4)[there]
    out = {"out": o.reshape(-1, qh * DIM).to(dt)}
    if case["weights"]:
        add = p.sum(dim=2)                                             # [n, kv_heads, L]
        pad = blocks * PAGE - L
        add = torch.nn.functional.pad(add, (0, pad)).reshape(n, kvh, blocks, PAGE).transpose(1, 2)
        st["weights"][st["table"][st["sids"].long(), :blocks].long()] += add
        out["weights"] = st["weights"]
    return out


def _plain_evict(st):
    case = st["case"]
    dt, kvh, n, keep, recent = (TYPES[case["dtype"]], case["kv_heads"], case["seqs"], case["keep"],
                                case["recent"])
    L, dev = st["max_len"], st["pages"].device
    blocks = -(-L // PAGE)
    rows = st["table"][st["sids"].long(), :blocks].long()
    flat = lambda t: t[rows].transpose(1, 2).reshape(n, kvh, blocks * PAGE)[..., :L]  # noqa: E731
    w, pos = flat(st["weights"]), flat(st["positions"])
    lens = st["lens"].long()
    slot = torch.arange(L, device=dev)
    there = (slot < lens[:, None])[:, None].expand(n, kvh, L)
    newest = torch.where(there, pos, torch.full_like(pos, -2 ** 31)).amax(dim=-1, keepdim=True)
    # order: there and protected, then by weight, then the lowest slot
    key = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w)
    key = torch.where(pos.long() > newest.long() - recent, torch.full_like(w, math.inf), key)
    key = torch.where(there, key, torch.full_like(w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(n, kvh, L, dtype=torch.bool, device=dev)
    kept.scatter_(2, order[..., :keep], True)
    kept &= there
    new = lens.clamp(max=keep)
    # slot d keeps its own entry, or takes the next kept one from beyond `keep`
    low = slot < keep
    hole = ~kept & low & there
    mover = kept & ~low
    source = slot.expand(n, kvh, L).clone()
    source[hole] = slot.expand(n, kvh, L)[mover]
    source = source[..., :keep]
    fine = (torch.arange(source.shape[-1], device=dev) < new[:, None])[:, None].expand_as(source)
    i, h, d = fine.nonzero(as_tuple=True)
    s = source[fine]
    sid = st["sids"].long()[i]
    src, dst = st["table"][sid, s // PAGE].long(), st["dst_table"][sid, d // PAGE].long()
    so, do = s % PAGE, d % PAGE
    for a, b, width in ((0, 1024, 64), (1024, 2048, 64), (2048, 2176, 8), (2176, 2304, 8)):
        got = st["pages"][..., a:b].reshape(-1, kvh, PAGE, width)[src, h, so]
        at = a + width * do[:, None] + torch.arange(width, device=dev)
        st["pages"][dst[:, None], h[:, None], at] = got
    for name in ("weights", "positions"):
        st[name][dst, h, do] = st[name][src, h, so]
    zero = torch.zeros_like(st["sids"])
    k, v = _get(st, st["dst_table"], st["sids"], zero, new, keep, dt)
    return {"lens": new.int(), "weights": st["weights"], "positions": st["positions"], "k": k, "v": v}


# ---------------------------------------------------- the framework's calls
def _own(st):
    if "dial-27b_b200" not in sys.path:
        sys.path.insert(0, "dial-27b_b200")
    from dial_b200 import kv4

    case, kept = st["case"], st["keep_by"]
    if "shape" not in kept:  # what a program keeps beside its cache
        kept["shape"] = kv4.make_shape(
            case["q_heads"], case["kv_heads"], st["table"].shape[1], st["pages"].shape[0],
            max_pos=st.get("max_pos", 0), eps=EPS, k_scale=st["k_scale"], v_scale=st["v_scale"],
            dtype=TYPES[case["dtype"]])
        kept["cache"] = kv4.Kv4Cache(st["pages"], st.get("weights"), st.get("positions"))
    sh, cache = kept["shape"], kept["cache"]
    if case["op"] == "append":
        q = kv4.kv4_append(sh, cache, st["qkv"], st["table"], st["sids"], st["slots"], st["at"],
                           q_norm_w=st.get("q_norm"), k_norm_w=st.get("k_norm"),
                           cos=st.get("cos"), sin=st.get("sin"))
        k, v = kv4.kv4_read(sh, cache, st["table"], st["sids"], st["ends"], 1, first=st["slots"])
        return {"q": q, "k": k, "v": v}
    if case["op"] == "attention":
        o = kv4.kv4_attention(sh, cache, st["q"], st["table"], st["sids"], st["lens"],
                              st["max_len"], q_starts=st["starts"], max_q=st["max_q"],
                              accumulate=case["weights"])
        return {"out": o, "weights": st["weights"]} if case["weights"] else {"out": o}
    new = kv4.kv4_evict(sh, cache, st["table"], st["sids"], st["lens"], st["max_len"],
                        case["keep"], case["recent"], dst_table=st["dst_table"])
    k, v = kv4.kv4_read(sh, cache, st["dst_table"], st["sids"], new, case["keep"])
    return {"lens": new, "weights": st["weights"], "positions": st["positions"], "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict}[op](state)


def work(case):
    qh, kvh, op = case["q_heads"], case["kv_heads"], case["op"]
    entry = kvh * 144                    # a slot's codes and scales, k and v
    if op == "append":                   # rows in, q out, slots written, read back, values out
        row = (qh + 2 * kvh) * 256 + qh * 256 + 2 * entry + kvh * 512
        return {"bytes": case["rows"] * row, "flops": case["rows"] * (qh + 2 * kvh) * DIM * 8}
    lens = _lengths(case)
    if op == "attention":
        qs = _queries(case, lens)
        pairs = sum(q * n - q * (q - 1) // 2 for q, n in zip(qs, lens))
        size = sum(lens) * (entry + 8 * kvh * bool(case["weights"])) + sum(qs) * qh * 512
        return {"bytes": size, "flops": 4 * DIM * qh * pairs}
    kept = sum(min(n, case["keep"]) for n in lens)
    # weights and positions ranked, entries moved, then read and their values written
    return {"bytes": sum(lens) * 8 * kvh + kept * (2 * entry + 8 * kvh + entry + kvh * 512),
            "flops": 0}


# ------------------------------------------------------------ in 64 bits
def _exact_values(pages, block, off, g_k, g_v):
    """k and v of slots (block, off) of every head, 64 bits, [slots, kv_heads, 128]."""
    out = []
    for codes_at, scales_at, g in ((0, 2048, g_k), (1024, 2176, g_v)):
        at = off[:, None] * 64 + codes_at + torch.arange(64, device=off.device)
        c = pages[block].gather(2, at[:, None].expand(-1, pages.shape[1], -1))
        at = off[:, None] * 8 + scales_at + torch.arange(8, device=off.device)
        s = pages[block].gather(2, at[:, None].expand(-1, pages.shape[1], -1)).int()
        # e4m3: 1 sign, 4 exponent (bias 7), 3 mantissa bits
        e, f = (s >> 3 & 15).double(), (s & 7).double()
        scale = torch.where(e == 0, f * 2.0 ** -9, torch.exp2(e - 7) * (1 + f / 8))
        scale = torch.where(s >= 128, -scale, scale) * g
        # e2m1: 1 sign, 2 exponent (bias 1), 1 mantissa bit
        n = torch.stack([c & 15, c >> 4], dim=3).flatten(2).int()
        e, f = (n >> 1 & 3).double(), (n & 1).double()
        x = torch.where(e == 0, f / 2, torch.exp2(e - 1) * (1 + f / 2))
        x = torch.where(n >= 8, -x, x)
        out.append(x * scale.repeat_interleave(16, dim=2))
    return out


def _exact_quantised(x, g):
    """What x, 64 bits [..., 128], stands for once cached: the nearest e2m1
    multiple of its group's e4m3 scale."""
    grp = x.unflatten(-1, (8, 16))
    top = grp.abs().amax(-1, keepdim=True) / 6 / g
    # nearest e4m3: steps of 2^(exponent - 3), ties to the even step
    step = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -6))) - 3)
    s = (torch.round(top / step) * step).clamp(max=448.0) * g
    a = torch.where(s > 0, grp.abs() / s, torch.zeros_like(grp))
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(grp) * (torch.round(a / step) * step).clamp(max=6.0) * s).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    dt, qh, kvh = TYPES[case["dtype"]], case["q_heads"], case["kv_heads"]
    table, pages = st["table"].long(), st["pages"]
    if case["op"] == "append":
        x = st["qkv"].double().unflatten(1, (-1, DIM))
        parts = [x[:, :qh], x[:, qh:qh + kvh]]
        if case["norm"]:
            at = st["at"].long()
            c, s = st["cos"].double()[at].unsqueeze(1), st["sin"].double()[at].unsqueeze(1)
            r = lambda t: t.to(dt).double()  # noqa: E731
            for i, w in ((0, st["q_norm"]), (1, st["k_norm"])):
                y = parts[i]
                y = r(r(y / r((y.pow(2).mean(-1, keepdim=True) + EPS).sqrt())) * w.double())
                lo, hi = y.chunk(2, dim=-1)
                parts[i] = torch.cat([r(r(lo * c) - r(hi * s)), r(r(hi * c) + r(lo * s))], -1)
        return {"q": parts[0].flatten(1), "k": _exact_quantised(parts[1], st["k_scale"])[:, None],
                "v": _exact_quantised(x[:, qh + kvh:], st["v_scale"])[:, None]}
    lens, sids = _lengths(case), st["sids"].tolist()
    if case["op"] == "attention":
        starts, rep = st["starts"].tolist(), qh // kvh
        out = torch.empty(starts[-1], qh, DIM, dtype=torch.float64, device=pages.device)
        acc = st["weights"].double()
        for i, (n, sid) in enumerate(zip(lens, sids)):
            slot = torch.arange(n, device=pages.device)
            block, off = table[sid, slot // PAGE], slot % PAGE
            k, v = _exact_values(pages, block, off, st["k_scale"], st["v_scale"])
            q = st["q"][starts[i]:starts[i + 1]].double().unflatten(1, (-1, DIM))
            late = slot[None] > n - q.shape[0] + torch.arange(q.shape[0], device=slot.device)[:, None]
            add = torch.zeros(n, kvh, dtype=torch.float64, device=slot.device)
            for h in range(qh):
                s = (q[:, h] @ k[:, h // rep].T) * DIM ** -0.5
                p = torch.softmax(s.masked_fill(late, -math.inf), dim=-1)
                out[starts[i]:starts[i + 1], h] = p @ v[:, h // rep]
                add[:, h // rep] += p.sum(0)
            acc[block, :, off] += add
        got = {"out": out.flatten(1)}
        if case["weights"]:
            got["weights"] = acc
        return got
    keep, recent, n = case["keep"], case["recent"], case["seqs"]
    dst = st["dst_table"].long()
    k_out = torch.zeros(n, keep, kvh, DIM, dtype=torch.float64, device=pages.device)
    v_out, acc = k_out.clone(), st["weights"].double()
    for i, (have, sid) in enumerate(zip(lens, sids)):
        slot = torch.arange(have, device=pages.device)
        block, off = table[sid, slot // PAGE], slot % PAGE
        k, v = _exact_values(pages, block, off, st["k_scale"], st["v_scale"])
        w = st["weights"][block, :, off].cpu().numpy()
        p = st["positions"][block, :, off].cpu().numpy().astype(np.int64)
        new = min(have, keep)
        for h in range(kvh):
            safe = p[:, h] > p[:, h].max() - recent
            best = np.lexsort((np.arange(have), -w[:, h].astype(np.float64), ~safe))[:new]
            stay = np.zeros(have, bool)
            stay[best] = True
            place = np.arange(new)
            place[~stay[:new]] = np.nonzero(stay[new:])[0] + new
            at = torch.from_numpy(place).to(pages.device)
            k_out[i, :new, h], v_out[i, :new, h] = k[at, h], v[at, h]
            d = slot[:new]
            acc[dst[sid, d // PAGE], h, d % PAGE] = torch.from_numpy(
                w[place, h].astype(np.float64)).to(pages.device)
    return {"lens": None, "weights": acc, "positions": None, "k": k_out, "v": v_out}
