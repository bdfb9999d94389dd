"""Plain 64-bit reference of the 4-bit KV cache operators, and random problems
for their tests: caches held as codes and scales in numpy, with the page layout
of include/dial_b200.h restated here."""

import numpy as np
import torch

PAGE, DIM, SLAB = 16, 128, 2304
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
E2M1 = np.concatenate([E2M1, -E2M1])
# every e4m3 value by code (0x7f / 0xff are NaN)
_c = np.arange(256)
_e, _m = _c >> 3 & 15, _c & 7
E4M3 = np.where(_e == 0, _m * 2.0 ** -9, 2.0 ** (_e - 7.0) * (1 + _m / 8))
E4M3 = np.where(_c >= 128, -E4M3, E4M3)
E4M3[[0x7F, 0xFF]] = np.nan


def act_round(x, dt):
    """Nearest value of the activation dtype, as float64."""
    return torch.from_numpy(np.asarray(x, np.float32)).to(dt).double().numpy()


def nearest(x, grid):
    """Index of the nearest of the rising `grid` (ties to the even index,
    saturating), for x >= 0."""
    hi = np.clip(np.searchsorted(grid, x), 0, len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    up = (x - grid[lo] > grid[hi] - x) | ((x - grid[lo] == grid[hi] - x) & (hi % 2 == 0))
    return np.where(up | (x >= grid[-1]), hi, lo)


def encode(x, mult):
    """x [..., 128] to codes [..., 128] and e4m3 scale codes [..., 8]."""
    x = np.where(np.isnan(x), 0.0, x).reshape(*x.shape[:-1], 8, 16)
    with np.errstate(invalid="ignore", over="ignore"):
        top = np.minimum(np.abs(x).max(-1) / 6 / mult, 448.0)
    sc = nearest(top, E4M3[:127])
    s = (E4M3[sc] * mult)[..., None]
    a = np.where(s > 0, np.abs(x) / np.where(s > 0, s, 1), 0)
    code = nearest(np.minimum(a, 6.0), E2M1[:8]) | (np.signbit(x) & (s > 0)) * 8
    return code.reshape(*code.shape[:-2], 128).astype(np.uint8), sc.astype(np.uint8)


def decode(code, sc, mult):
    v = E2M1[code].reshape(*code.shape[:-1], 8, 16) * (E4M3[sc] * mult)[..., None]
    return v.reshape(code.shape)


def pack(k, ks, v, vs):
    """Codes [..., 16, 128] and scales [..., 16, 8] to slabs [..., 2304]."""
    nib = lambda c: (c[..., 0::2] | c[..., 1::2] << 4).reshape(*c.shape[:-2], 1024)  # noqa: E731
    flat = lambda s: s.reshape(*s.shape[:-2], 128)  # noqa: E731
    return np.concatenate([nib(k), nib(v), flat(ks), flat(vs)], axis=-1)


def unpack(slab):
    def nib(b):
        b = b.reshape(*b.shape[:-1], 16, 64)
        return np.stack([b & 15, b >> 4], axis=-1).reshape(*b.shape[:-1], 128)
    r = lambda b: b.reshape(*b.shape[:-1], 16, 8)  # noqa: E731
    return nib(slab[..., :1024]), r(slab[..., 2048:2176]), nib(slab[..., 1024:2048]), r(
        slab[..., 2176:])


def norm_rope(x, w, cos, sin, eps, dt):
    """Rows [rows, heads, 128]: RMSNorm (w) and RoPE (cos, sin [rows, 64]),
    each step rounded to dt."""
    r = lambda t: act_round(t, dt)  # noqa: E731
    if w is not None:
        m = r(np.sqrt(np.mean(x * x, -1, keepdims=True) + eps))
        x = r(r(x / m) * w)
    if cos is not None:
        a, b, c, s = x[..., :64], x[..., 64:], cos[:, None], sin[:, None]
        x = np.concatenate([r(r(a * c) - r(b * s)), r(r(a * s) + r(b * c))], -1)
    return x


class Cache:
    """A pool, its tables and its tracked arrays, on the host."""

    def __init__(self, seed, sessions, capacity, q_heads, kv_heads, dt=torch.bfloat16,
                 k_scale=0.5, v_scale=0.0625, spare=2, fill=True, max_pos=0):
        from dial_b200 import kv4

        self.rng = np.random.default_rng(seed)
        self.QH, self.H, self.dt = q_heads, kv_heads, dt
        self.rep = q_heads // kv_heads
        self.max_blocks = -(-capacity // PAGE)
        nb = sessions * self.max_blocks + spare
        self.table = self.rng.permutation(nb)[:sessions * self.max_blocks].astype(np.int32).reshape(
            sessions, self.max_blocks)
        self.k_scale, self.v_scale = k_scale, v_scale
        r = self.rng.standard_normal
        chan = np.exp(0.5 * r((kv_heads, 1, DIM)))
        if fill:
            self.pages = pack(*encode(r((nb, kv_heads, PAGE, DIM)) * chan, k_scale),
                              *encode(r((nb, kv_heads, PAGE, DIM)) * 0.5, v_scale))
        else:
            self.pages = self.rng.integers(0, 256, (nb, kv_heads, SLAB)).astype(np.uint8)
            self.pages[..., 2048:] &= 0x77  # finite scales
        self.weights = np.exp(r((nb, kv_heads, PAGE))).astype(np.float32)
        self.positions = self.rng.integers(0, 1 << 20, (nb, kv_heads, PAGE)).astype(np.int32)
        self.sh = kv4.make_shape(q_heads, kv_heads, self.max_blocks, nb, max_pos=max_pos,
                                 k_scale=k_scale, v_scale=v_scale, dtype=dt)

    def device(self, cuda):
        from dial_b200 import kv4

        t = lambda a: torch.from_numpy(a.copy()).to(cuda)  # noqa: E731
        return kv4.Kv4Cache(t(self.pages), t(self.weights), t(self.positions)), t(self.table)

    def at(self, sid, n):
        slot = np.arange(n)
        return self.table[sid, slot // PAGE], slot % PAGE

    def values(self, sid, n):
        """k and v [n, kv_heads, 128] of the session's slots."""
        k, ks, v, vs = unpack(self.pages[self.table[sid, :-(-n // PAGE)]])  # [pages, heads, 16, .]
        flat = lambda x: x.transpose(0, 2, 1, 3).reshape(-1, self.H, x.shape[-1])[:n]  # noqa: E731
        return (decode(flat(k), flat(ks), self.k_scale), decode(flat(v), flat(vs), self.v_scale))

    def put(self, sid, slot, k, v, pos):
        """One token's k and v [kv_heads, 128] into its slot."""
        b, o = self.table[sid, slot // PAGE], slot % PAGE
        slabs = [x.copy() for x in unpack(self.pages[b])]
        for i, (x, g) in enumerate(((k, self.k_scale), (v, self.v_scale))):
            slabs[2 * i][:, o], slabs[2 * i + 1][:, o] = encode(x, g)
        self.pages[b] = pack(*slabs)
        self.weights[b, :, o] = 0
        if pos is not None:
            self.positions[b, :, o] = pos

    def attend(self, q, sid, n, scale=DIM ** -0.5):
        """(out [rows, QH * 128], its error bound, slot sums [n, kv_heads], their
        bound) of the queries q [rows, QH * 128] at the end of n slots.

        Bounds, from the roundings of any evaluation with 32-bit scores, sums
        and accumulators and probabilities of at least 11 bits: a score is off by
        at most 2^-19 of scale * sum |q k| (128 products accumulated in f32, each
        step truncated at worst, twice for the two chains) plus 2^-20 for the
        exponent's own rounding, its probability by twice that relative, once
        more for the sum l; a probability in f16 by 2^-11 relative or 2^-25 of the
        largest absolute; the f32 sums of n terms by n * 2^-24 but no more than 2^-10;
        the output's rounding is half a step of its dtype."""
        rows = q.shape[0]
        K, V = self.values(sid, n)
        Q = q.reshape(rows, self.QH, DIM)
        out, bound = np.zeros((rows, self.QH, DIM)), np.zeros((rows, self.QH, DIM))
        sums, sbound = np.zeros((n, self.H)), np.zeros((n, self.H))
        half = torch.finfo(self.dt).eps / 2
        for j in range(rows):
            seen = n - rows + 1 + j
            if seen <= 0:
                continue
            for h in range(self.QH):
                g = h // self.rep
                k, v = K[:seen, g], V[:seen, g]
                s = (k @ Q[j, h]) * scale
                off = 2.0 ** -19 * (np.abs(k) @ np.abs(Q[j, h])).max() * scale + 2.0 ** -20
                p = np.exp(s - s.max())
                p /= p.sum()
                o = p @ v
                rel = 4 * off + min(seen * 2.0 ** -24, 2.0 ** -10)
                err = (rel + 2.0 ** -11) * (p @ np.abs(v)) + seen * 2.0 ** -25 * np.abs(v).max()
                tiny = 2.0 ** -24 if self.dt == torch.float16 else 2.0 ** -126
                out[j, h], bound[j, h] = o, err + half * (np.abs(o) + err) + tiny
                sums[:seen, g] += p
                sbound[:seen, g] += p * rel
        width = self.QH * DIM
        return out.reshape(rows, width), bound.reshape(rows, width), sums, sbound + 2.0 ** -22 * sums

    def evict(self, sid, n, keep, recent, dst=None):
        """Cut one session; the new length.  `dst`: table to move into."""
        dst = self.table if dst is None else dst
        new = min(n, keep)
        b, o = self.at(sid, n)
        old = {x: getattr(self, x)[b, :, o].copy() for x in ("weights", "positions")}
        parts = [x[b, :, o].copy() for x in unpack(self.pages)]
        for h in range(self.H):
            w, p = old["weights"][:, h], old["positions"][:, h].astype(np.int64)
            safe = p > p.max(initial=-2 ** 31) - recent if recent > 0 else np.zeros(n, bool)
            best = sorted(range(n), key=lambda i: (
                not safe[i], bool(np.isnan(w[i])), 0 if np.isnan(w[i]) else -float(w[i]), i))[:new]
            stay = np.zeros(n, bool)
            stay[best] = True
            src = np.arange(new)
            src[~stay[:new]] = np.nonzero(stay[new:])[0] + new
            for d, s in enumerate(src):
                tb, to = dst[sid, d // PAGE], d % PAGE
                slabs = [x.copy() for x in unpack(self.pages[tb, h])]
                for part, x in zip(slabs, parts):
                    part[to] = x[s, h]
                self.pages[tb, h] = pack(*slabs)
                self.weights[tb, h, to] = old["weights"][s, h]
                self.positions[tb, h, to] = old["positions"][s, h]
        return new


def same_slabs(got, want):
    """Bitwise equal but for the sign of a zero code."""
    a, b = unpack(got), unpack(want)
    for x, y in zip(a[0::2], b[0::2]):
        np.testing.assert_array_equal(np.where(x == 8, 0, x), np.where(y == 8, 0, y))
    for x, y in zip(a[1::2], b[1::2]):
        np.testing.assert_array_equal(x, y)


def i32(cuda, *v):
    return torch.tensor(v, dtype=torch.int32, device=cuda)
