"""What the tests of the paged K/V cache share: its definition in numpy, in 64 bits and apart from the kernels, and a
cache in device buffers beside it."""
import numpy as np

import moert

B = moert.PAGES_BLOCK
F32, F16, BF16 = moert.F32, moert.F16, moert.BF16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step of the type, relative
INF = {F16: 0x7C00, BF16: 0x7F80}  # bits from which a 16-bit value is not finite


def to_bits(x, dtype):
    """f32 values as rows of a type: f32 itself, or the 16 bits of the nearest value (ties to even)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == F32:
        return x
    if dtype == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    w = x.view(np.uint32).astype(np.uint64)
    r = ((w + 0x7FFF + (w >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FFF), r)


def from_bits(b, dtype):
    """Rows of a type as 64-bit values."""
    if dtype == F32:
        return b.astype(np.float64)
    if dtype == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def k_place(t, e):
    return ((e // 8) * 32 + t) * 8 + e % 8


def v_place(t, e, d):
    return ((t // 16 * 2 + t % 8 // 4) * d + e) * 8 + t % 4 + 4 * (t % 16 // 8)


class Cache:
    """The cache from its definition: pages of each sequence, free pages, and the rows that lie in the pool."""

    def __init__(self, seqs, kv_heads, d, page, pages, max_pages, dtype=F16):
        self.S, self.H, self.d, self.P, self.N, self.M, self.dtype = seqs, kv_heads, d, page, pages, max_pages, dtype
        self.free = list(range(pages - 1, -1, -1))
        self.table = [[] for _ in range(seqs)]
        self.rows, self.refused, self.first = [0] * seqs, [0] * seqs, [0] * seqs
        self.k = np.full((pages * page, kv_heads, d), np.nan)  # by slot; NaN: never written
        self.v = np.full((pages * page, kv_heads, d), np.nan)

    def plan(self, new, tokens):
        """starts, slots, positions."""
        for s, n in enumerate(new):
            if n < 0:
                self.free += self.table[s]
                self.table[s], self.rows[s], self.refused[s], self.first[s] = [], 0, 0, 0
        starts, slots, positions, short = [0], [], [], False
        for s, n in enumerate(max(int(x), 0) for x in new):
            rows = self.rows[s]
            need = -(-(rows + n) // self.P) - -(-rows // self.P)
            ok = n == 0 or (starts[-1] + n <= tokens and rows + n <= self.M * self.P)
            if ok and need and (short or need > len(self.free)):
                ok, short = False, True
            if ok:
                self.table[s] += [self.free.pop() for _ in range(need)]
                at = range(rows, rows + n)
                slots += [self.table[s][p // self.P] * self.P + p % self.P for p in at]
                positions += list(at)
                self.rows[s] = rows + n
            else:
                self.refused[s] = min(self.refused[s] + n, 2 ** 31 - 1)
                room = min(n, tokens - starts[-1])
                slots += [-1] * room
                positions += [-1] * room
            self.first[s] = rows if ok else -1
            starts.append(starts[-1] + (n if ok else min(n, tokens + 1 - starts[-1])))
        pad = [-1] * (tokens - len(slots))
        return (np.minimum(starts, tokens).astype(np.int32), np.array(slots + pad, np.int32),
                np.array(positions + pad, np.int32))

    def append(self, k, v, slots, dtype):
        """k, v: rows of `dtype`, as to_bits gives them; poisoned rows become NaN."""
        for i, slot in enumerate(slots):
            if 0 <= slot < self.N * self.P:
                kk, vv = (from_bits(to_bits(from_bits(x[i], dtype), self.dtype), self.dtype) for x in (k, v))
                bad = ~(np.isfinite(kk).all(1) & np.isfinite(vv).all(1))
                kk[bad] = vv[bad] = np.nan
                self.k[slot], self.v[slot] = kk, vv

    def seen(self, s):
        return 0 if self.first[s] < 0 else self.rows[s]

    def kv(self, s, h, n):
        at = np.arange(n)
        slots = np.array(self.table[s], np.int64)[at // self.P] * self.P + at % self.P if n else at
        return self.k[slots, h], self.v[slots, h]

    def attend(self, q, starts, scale, out_type, which=lambda n: True):
        """q [tokens, heads, d] in 64 bits -> outputs, bounds of their error, and which rows are written. A bound is
        0 where the output is 0 or NaN.

        A score is a sum of d products. Queries of f32 enter as two fp16, off by 2^-22 of an element, 16-bit ones as
        they are; sums in f32 lose at most 2^-23 of the sum of magnitudes per addition, d + 8 of them with the scales'
        products. So a score is off by E = scale sum|q k| ((d + 8) 2^-23 + 2^-22), a weight by the factor exp(2 E) (its
        own score's and the sum's). exp2 is good to 2 ulp, on arguments of up to 1.5 max|s| + 32: 2^-22 of (1.5 max|s| +
        32). Sums of weights and products: 2^-23 per block and 64 beside. Weights of the second product are rounded to
        half a step of the cache's type (16-bit outputs), or 2^-21 as two numbers, and to 2^-24 of the largest. The sum
        may hold them before that rounding: twice. Outputs are rounded once more."""
        tokens, heads, d = q.shape
        g = heads // self.H
        out, off, wrote = np.zeros(q.shape), np.zeros(q.shape), np.zeros(tokens, bool)
        for s in range(self.S):
            lo, hi = int(starts[s]), int(starts[s + 1])
            n, L = hi - lo, self.seen(s)
            if not n or not which(n):
                continue
            wrote[lo:hi] = True
            for i in range(n):
                m = L - n + 1 + i
                if m <= 0:
                    continue
                for a in range(heads):
                    x = q[lo + i, a]
                    k, v = self.kv(s, a // g, m)
                    if not (np.isfinite(k).all() and np.isfinite(x).all()):
                        out[lo + i, a] = np.nan
                        continue
                    sc = scale * (k @ x)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    mag = abs(scale) * (np.abs(k) @ np.abs(x)).max()
                    e = 2 * mag * ((d + 8) * 2.0 ** -23 + 2.0 ** -22) + (1.5 * np.abs(sc).max() + 32) * 2.0 ** -22 + \
                        (64 + 4 * -(-m // B)) * 2.0 ** -23
                    r = e + (2.0 ** -21 if out_type == F32 else 2 * HALF[self.dtype])
                    out[lo + i, a] = p @ v
                    off[lo + i, a] = r * (p @ np.abs(v)) + m * 2.0 ** -24 * p.max() * np.abs(v).max() + \
                        HALF[out_type] * np.abs(p @ v) + (2.0 ** -24 if out_type == F16 else 0.0)
        return out, off, wrote


class Device:
    """A cache in device buffers, beside moert.Pages; memory that nothing has written holds NaN and -1."""

    def __init__(self, hip, seqs, kv_heads, d, page, pages, max_pages, dtype=F16, fill=True):
        self.hip, self.d, self.dtype = hip, d, dtype
        self.shapes = moert.pages_shapes(seqs, kv_heads, d, page, pages, max_pages)
        self.at = {}
        for name, (shape, t) in self.shapes.items():
            n = int(np.prod(shape)) * np.dtype(t).itemsize
            self.at[name] = hip.upload(np.full(n, 0xFF, np.uint8)) if fill else hip.alloc(n)
        self.c = moert.Pages(seqs, kv_heads, d, page, pages, max_pages, self.at, dtype=dtype)
        self.c.clear()

    def array(self, name):
        self.hip.sync()
        return self.hip.get(self.at[name], *self.shapes[name])

    def set(self, name, a):
        self.hip.put(self.at[name], np.ascontiguousarray(a, self.shapes[name][1]).reshape(self.shapes[name][0]))

    def plan(self, new, tokens, stream=0, positions=True):
        """starts, slots, positions, and their addresses."""
        S, hip = self.c.seqs, self.hip
        at = [hip.upload(np.full(max(n, 1), 77, np.int32)) for n in (S + 1, tokens, tokens)]
        self.c.plan(hip.upload(np.asarray(new, np.int32)), tokens, at[0], at[1] if tokens else 0,
                    at[2] if positions else 0, stream=stream)
        hip.sync()
        got = [hip.get(p, (n,), np.int32) for p, n in zip(at, (S + 1, tokens, tokens))]
        return got, at

    def append(self, k, v, slots, dtype, **kw):
        """slots: an address, or values."""
        at = slots if isinstance(slots, int) else self.hip.upload(np.asarray(slots, np.int32))
        self.c.append(self.hip.upload(k), self.hip.upload(v), at, k.shape[0], dtype=dtype, **kw)

    def workspace(self, heads, tokens=0):
        size = self.c.workspace(heads, tokens)
        return self.hip.upload(np.full(max(size, 16), 0xFF, np.uint8)), size

    def _out(self, q, dtype):
        return self.hip.upload(np.full(q.shape, 7.0, np.float32) if dtype == F32 else np.full(q.shape, 0x4321, np.uint16))

    def attend(self, q, scale, dtype, starts=None, **kw):
        """q as to_bits gives it; starts as values."""
        out = self._out(q, dtype)
        ws, size = self.workspace(q.shape[1])
        at = 0 if starts is None else self.hip.upload(np.asarray(starts, np.int32))
        self.c.attend(self.hip.upload(q), out, q.shape[1], scale, ws, size, starts=at, tokens=q.shape[0], dtype=dtype, **kw)
        self.hip.sync()
        return self.hip.get(out, q.shape, q.dtype)

    def prompt(self, q, scale, dtype, starts, **kw):
        out = self._out(q, dtype)
        ws, size = self.workspace(q.shape[1], q.shape[0])
        self.c.prompt(self.hip.upload(q), out, q.shape[1], scale, self.hip.upload(np.asarray(starts, np.int32)),
                      q.shape[0], ws, size, dtype=dtype, **kw)
        self.hip.sync()
        return self.hip.get(out, q.shape, q.dtype)


def untouched(dtype):
    return np.float32(7.0) if dtype == F32 else np.uint16(0x4321)


def assert_planned(dev, ref):
    """The device's state, tables and free pages are the definition's."""
    state, table, free = (dev.array(n) for n in ("state", "table", "free"))
    assert state[:, 0].tolist() == ref.rows
    assert state[:, 1].tolist() == ref.refused
    assert state[:, 2].tolist() == ref.first
    assert free[0] == len(ref.free) and free[1:1 + len(ref.free)].tolist() == ref.free
    for s, pages in enumerate(ref.table):
        assert table[s, :len(pages)].tolist() == pages, s


def assert_holds(dev, ref):
    """The pool holds the definition's rows, bit for bit: a poisoned row a K of NaN and a V of 0, memory that was never
    written as it was."""
    t, e = np.arange(B)[:, None], np.arange(ref.d)[None, :]
    for name, place, want in (("k", k_place(t, e), ref.k), ("v", v_place(t, e, ref.d), ref.v)):
        got = dev.array(name)[..., place]  # [pages, H, blocks, B, d]
        got = got.transpose(0, 2, 3, 1, 4).reshape(want.shape)
        bits = to_bits(want.astype(np.float32), ref.dtype)
        bad = np.isnan(want).any(2)
        assert np.array_equal(got[~bad], bits[~bad]), name
        left = bad & (got == 0xFFFF).all(2)  # never written: as it was
        poisoned = bad & ~left
        if name == "k":
            assert ((got[poisoned] & 0x7FFF) > INF[ref.dtype]).all()
        else:
            assert not got[poisoned].any()


def check(got, want, q_type, wrote=None):
    """Outputs of a type against (outputs, bounds, which rows): NaN where NaN is due, 0 where nothing is seen, rows that
    are left out as they were."""
    out, off, rows = want
    assert (got[~rows] == untouched(q_type)).all()
    x = from_bits(got, q_type)
    assert np.array_equal(np.isnan(x[rows]), np.isnan(out[rows]))
    fine = rows[:, None, None] & ~np.isnan(out)
    err, lim = np.abs(x - out)[fine], off[fine]
    assert (err <= lim).all(), f"{(err / np.maximum(lim, 1e-300)).max()} of its bound"
