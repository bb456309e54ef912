"""What the tests of the 8-bit K/V cache share: its definition in numpy, in 64 bits and apart from the kernels, and
device buffers of the HIP runtime that the library is linked against (libamdhip64.so.7), so that one runtime serves the
process."""
import ctypes

import numpy as np

import moert

B = moert.KV8_BLOCK


class Hip:
    """Buffers, streams, captures."""

    H2D, D2H, D2D = 1, 2, 3

    def __init__(self):
        moert.lib()
        rt = self.rt = ctypes.CDLL("libamdhip64.so.7")
        vp, sz = ctypes.c_void_p, ctypes.c_size_t
        rt.hipMalloc.argtypes = [ctypes.POINTER(vp), sz]
        rt.hipMemcpy.argtypes = [vp, vp, sz, ctypes.c_int]
        rt.hipFree.argtypes = [vp]
        rt.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(vp), ctypes.c_uint]
        rt.hipStreamSynchronize.argtypes = [vp]
        rt.hipStreamDestroy.argtypes = [vp]
        rt.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
        rt.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
        rt.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, sz]
        rt.hipGraphLaunch.argtypes = [vp, vp]
        rt.hipGraphExecDestroy.argtypes = [vp]
        rt.hipGraphDestroy.argtypes = [vp]
        self.bufs, self.streams, self.graphs = [], [], []

    def check(self, rc):
        assert rc == 0, f"HIP error {rc}"

    def alloc(self, nbytes: int) -> int:
        p = ctypes.c_void_p()
        self.check(self.rt.hipMalloc(ctypes.byref(p), max(nbytes, 16)))
        self.bufs.append(p)
        return p.value

    def put(self, at: int, a: np.ndarray):
        a = np.ascontiguousarray(a)
        self.check(self.rt.hipMemcpy(at, a.ctypes.data, a.nbytes, self.H2D))

    def upload(self, a: np.ndarray) -> int:
        at = self.alloc(a.nbytes)
        self.put(at, a)
        return at

    def get(self, at: int, shape, dtype) -> np.ndarray:
        a = np.empty(shape, dtype)
        self.check(self.rt.hipMemcpy(a.ctypes.data, at, a.nbytes, self.D2H))
        return a

    def sync(self):
        self.check(self.rt.hipDeviceSynchronize())

    def stream(self) -> int:
        s = ctypes.c_void_p()
        self.check(self.rt.hipStreamCreateWithFlags(ctypes.byref(s), 1))
        self.streams.append(s)
        return s.value

    def capture(self, stream: int, calls):
        """The calls on the stream as an executable graph."""
        g, x = ctypes.c_void_p(), ctypes.c_void_p()
        self.check(self.rt.hipStreamBeginCapture(stream, 1))
        calls()
        self.check(self.rt.hipStreamEndCapture(stream, ctypes.byref(g)))
        self.check(self.rt.hipGraphInstantiate(ctypes.byref(x), g, None, None, 0))
        self.graphs.append((g, x))
        return x

    def launch(self, graph, stream: int):
        self.check(self.rt.hipGraphLaunch(graph, stream))

    def close(self):
        self.rt.hipDeviceSynchronize()
        for g, x in self.graphs:
            self.rt.hipGraphExecDestroy(x)
            self.rt.hipGraphDestroy(g)
        for s in self.streams:
            self.rt.hipStreamDestroy(s)
        for p in self.bufs:
            self.rt.hipFree(p)
        self.bufs, self.streams, self.graphs = [], [], []


# ---- the definition ------------------------------------------------------------------------------------------------
def v_place(t, e, d):
    """Place of position t, element e in a block of V."""
    u = d // 16
    return ((e // u * 4 + t % 16 // 4) * u + e % u) * 8 + t % 4 + 4 * (t // 16)


def v_order(d):
    """[32, d] places of a block of V."""
    return v_place(np.arange(B)[:, None], np.arange(d)[None, :], d)


def code_block(x):
    """x [32, d] fp16: (codes as integers, scale f32)."""
    x = x.astype(np.float64)
    if not np.isfinite(x).all():
        return np.zeros(x.shape, np.int64), np.float32(np.nan)
    a = np.abs(x).max()
    s = np.float32(np.float32(a) / np.float32(127.0)) if a else np.float32(1.0)
    return np.rint(x / np.float64(s)).astype(np.int64), s


class Cache:
    """The cache from its definition: per sequence and head a list of blocks (codes k, scale k, codes v, scale v,
    mass) and the tail's rows in fp16 with its mass."""

    def __init__(self, seqs, kv_heads, d, max_len):
        self.S, self.H, self.d, self.max_len = seqs, kv_heads, d, max_len
        self.blocks = [[[] for _ in range(kv_heads)] for _ in range(seqs)]
        self.tail = [[(np.zeros((0, d), np.float16),) * 2 for _ in range(kv_heads)] for _ in range(seqs)]
        self.tail_mass = np.zeros((seqs, kv_heads))
        self.dropped = [0] * seqs

    def len(self, s):
        return B * len(self.blocks[s][0]) + len(self.tail[s][0][0])

    def append(self, k, v, seq0=0):
        """k, v [n_seqs, n, H, d]."""
        with np.errstate(over="ignore"):
            k, v = k.astype(np.float16), v.astype(np.float16)
        for i in range(k.shape[0]):
            s, n = seq0 + i, k.shape[1]
            if self.len(s) + n > self.max_len:
                self.dropped[s] += n
                continue
            for h in range(self.H):
                rows = [np.concatenate([self.tail[s][h][p], (k, v)[p][i, :, h]]) for p in (0, 1)]
                while len(rows[0]) >= B:
                    (ck, sk), (cv, sv) = code_block(rows[0][:B]), code_block(rows[1][:B])
                    self.blocks[s][h].append([ck, sk, cv, sv, self.tail_mass[s, h]])
                    self.tail_mass[s, h] = 0.0
                    rows = [r[B:] for r in rows]
                self.tail[s][h] = tuple(rows)

    def rows(self, s, h):
        """K, V [len, d] in 64 bits, NaN for what is not finite; and whether a position is poisoned."""
        k = [b[0] * np.float64(b[1]) for b in self.blocks[s][h]]
        v = [b[2] * np.float64(b[3]) for b in self.blocks[s][h]]
        bad = [np.full(B, np.isnan(b[1]) or np.isnan(b[3])) for b in self.blocks[s][h]]
        tk, tv = (x.astype(np.float64) for x in self.tail[s][h])
        bad.append(~(np.isfinite(tk).all(1) & np.isfinite(tv).all(1)))
        return np.concatenate(k + [tk]), np.concatenate(v + [tv]), np.concatenate(bad)

    def attend(self, q, scale, decay=None, seq0=0):
        """q [n_seqs, n, heads, d] -> out in 64 bits; with decay the masses move on."""
        q = q.astype(np.float64)
        N, n, heads, d = q.shape
        g = heads // self.H
        out = np.zeros(q.shape)
        for i in range(N):
            s = seq0 + i
            L = self.len(s)
            for h in range(self.H):
                k, v, bad = self.rows(s, h)
                w = np.zeros(-(-L // B) * B)
                for j in range(n):
                    m = L - n + 1 + j
                    if m <= 0:
                        continue
                    for a in range(h * g, h * g + g):
                        if bad[:m].any():
                            out[i, j, a] = np.nan
                            w[:m] = np.nan
                            continue
                        x = scale * (k[:m] @ q[i, j, a])
                        p = np.exp(x - x.max())
                        p /= p.sum()
                        out[i, j, a] = p @ v[:m]
                        w[:m] += p
                if decay is not None:
                    w = w.reshape(-1, B).sum(1)
                    for b, blk in enumerate(self.blocks[s][h]):
                        blk[4] = decay * blk[4] + w[b]
                    if L % B:
                        self.tail_mass[s, h] = decay * self.tail_mass[s, h] + w[-1]
        return out

    def evict(self, keep, first, last, seq0=0, n_seqs=None):
        for s in range(seq0, self.S if n_seqs is None else seq0 + n_seqs):
            for h in range(self.H):
                blocks = self.blocks[s][h]
                nb = len(blocks)
                if nb <= keep:
                    continue
                may = range(first, nb - last)
                best = sorted(may, key=lambda b: (-np.inf if np.isnan(blocks[b][4]) else -blocks[b][4], b))
                if any(np.isnan(b[4]) for b in blocks):
                    best = sorted(may, key=lambda b: (0, 0, b) if np.isnan(blocks[b][4]) else (1, -blocks[b][4], b))
                stay = set(best[:keep - first - last]) | set(range(first)) | set(range(nb - last, nb))
                self.blocks[s][h] = [x for b, x in enumerate(blocks) if b in stay]

    def read(self, s, pos, n):
        """K, V [n, H, d] in 64 bits, 0 where there is no position; poisoned blocks NaN, the tail as it is."""
        k, v = np.zeros((n, self.H, self.d)), np.zeros((n, self.H, self.d))
        L = self.len(s)
        first = L + pos if pos < 0 else pos
        for h in range(self.H):
            a, b, _ = self.rows(s, h)
            for i in range(n):
                if 0 <= first + i < L:
                    k[i, h], v[i, h] = a[first + i], b[first + i]
        return k, v


class Device:
    """A cache in device buffers, beside moert.Kv8: uploads, workspaces, what the buffers hold as the definition's."""

    def __init__(self, hip, seqs, kv_heads, d, max_len, fill=True):
        """fill: with random bytes, as whatever was there before; without, large buffers stay as they come."""
        self.hip, self.d = hip, d
        self.shapes = moert.kv8_shapes(seqs, kv_heads, d, max_len)
        rng = np.random.default_rng(5)
        self.at = {}
        for name, (shape, dtype) in self.shapes.items():  # whatever was there before: clear makes it a cache
            n = int(np.prod(shape)) * np.dtype(dtype).itemsize
            self.at[name] = hip.upload(rng.integers(0, 256, n, dtype=np.uint8)) if fill else hip.alloc(n)
        self.c = moert.Kv8(seqs, kv_heads, d, max_len, self.at)
        self.c.clear()
        self.ws = {}

    def append(self, k, v, dtype=moert.F32, **kw):
        t = np.float32 if dtype == moert.F32 else np.float16
        with np.errstate(over="ignore"):
            self.c.append(self.hip.upload(k.astype(t)), self.hip.upload(v.astype(t)), k.shape[1], dtype=dtype,
                          n_seqs=k.shape[0], **kw)

    def workspace(self, heads, n, n_seqs, track):
        key = (heads, n, n_seqs, track)
        if key not in self.ws:
            size = self.c.workspace(heads, n, n_seqs=n_seqs, track=track)
            self.ws[key] = (self.hip.upload(np.full(max(size, 16), 0xFF, np.uint8)), size)  # NaN, -1 all over
        return self.ws[key]

    def attend(self, q, scale, dtype=moert.F32, decay=None, **kw):
        t = np.float32 if dtype == moert.F32 else np.float16
        out = self.hip.upload(np.full(q.shape, 7.0, t))
        ws, size = self.workspace(q.shape[2], q.shape[1], q.shape[0], decay is not None)
        self.c.attend(self.hip.upload(q.astype(t)), out, q.shape[2], q.shape[1], scale, ws, size, dtype=dtype,
                      mass_decay=decay, n_seqs=q.shape[0], **kw)
        self.hip.sync()
        return self.hip.get(out, q.shape, t)

    def read(self, pos, n, dtype=moert.F32, n_seqs=None):
        t = np.float32 if dtype == moert.F32 else np.float16
        shape = (n_seqs or self.c.seqs, n, self.c.kv_heads, self.d)
        k, v = (self.hip.upload(np.full(shape, 7.0, t)) for _ in range(2))
        self.c.read(k, v, pos, n, dtype=dtype, n_seqs=n_seqs)
        self.hip.sync()
        return self.hip.get(k, shape, t), self.hip.get(v, shape, t)

    def array(self, name):
        self.hip.sync()
        shape, dtype = self.shapes[name]
        return self.hip.get(self.at[name], shape, dtype)

    def set(self, name, a):
        self.hip.put(self.at[name], a.astype(self.shapes[name][1]))

    def mass(self, s, h, blocks):
        """Masses of the first blocks, in order."""
        return self.array("mass")[s, h][self.array("table")[s, h, :blocks]]


def assert_holds(dev, ref):
    """The device's buffers hold what the definition says, bit for bit: codes, scales, tails, lengths, poison, table a
    permutation, and no mass outside the blocks in use."""
    a = {name: dev.array(name) for name in dev.shapes}
    order = v_order(dev.d).reshape(-1)
    for s in range(ref.S):
        assert a["state"][s].tolist() == [ref.len(s), ref.dropped[s], 0, 0], (s, a["state"][s])
        for h in range(ref.H):
            table, nb = a["table"][s, h], len(ref.blocks[s][h])
            assert sorted(table.tolist()) == list(range(table.size)), (s, h)
            for b, (ck, sk, cv, sv, _) in enumerate(ref.blocks[s][h]):
                assert np.array_equal(a["k_codes"][s, h, table[b]].astype(np.int64) - 128, ck), (s, h, b)
                got = a["v_codes"][s, h, table[b]].reshape(-1)[order].reshape(cv.shape).astype(np.int64) - 128
                assert np.array_equal(got, cv), (s, h, b)
                for name, want in (("k_scale", sk), ("v_scale", sv)):
                    have = a[name][s, h, table[b]]
                    assert have == want or (np.isnan(have) and np.isnan(want)), (s, h, b, name, have, want)
            r = len(ref.tail[s][h][0])
            kt = a["k_tail"][s, h].view(np.float16)
            vt = a["v_tail"][s, h].reshape(-1)[order].reshape(B, dev.d).view(np.float16)
            for got, want in ((kt[:r], ref.tail[s][h][0]), (vt[:r], ref.tail[s][h][1])):
                assert np.array_equal(got, want, equal_nan=True), (s, h)
            bad = 0
            for t in range(r):
                if not (np.isfinite(kt[t].astype(np.float64)).all() and np.isfinite(vt[t].astype(np.float64)).all()):
                    bad |= 1 << t
            assert int(a["tail_bad"][s, h]) & ((1 << r) - 1) == bad, (s, h)
            used = nb + (1 if r else 0)
            assert not a["mass"][s, h][table[used:]].any(), (s, h)
