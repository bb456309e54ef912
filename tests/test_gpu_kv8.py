"""The 8-bit K/V cache on the device against its definition in 64 bits (tests/kv8_util.py): what the cache holds bit for
bit, attention within bounds that follow from its roundings, evictions exactly."""
import numpy as np
import pytest

import kv8_util as ku
import moert

pytestmark = pytest.mark.gpu
B = ku.B


@pytest.fixture()
def hip(gpu):
    h = ku.Hip()
    yield h
    h.close()


def both(hip, seqs, kv_heads, d, max_len):
    return ku.Device(hip, seqs, kv_heads, d, max_len), ku.Cache(seqs, kv_heads, d, max_len)


def normal(rng, *shape, scale=1.0):
    return (scale * rng.standard_normal(shape)).astype(np.float32)


def out_bound(ref, q, scale, f16, seq0=0):
    """How far an output may be from the 64-bit one, and how far a block's weight, relative to it.

    A score is a sum of d products of q and k. q enters as two fp16 (F32: 22 bits, 2^-22 of an element) or exactly (F16);
    sums in f32 lose at most 2^-23 of the sum of magnitudes per addition, d + 8 of them with the scales' products. So a
    score is off by E = scale sum|q k| ((d + 8) 2^-23 + 2^-22), a weight by the factor exp(2 E) (its own score's and the
    sum's). exp2 and log2 are good to 2 ulp, on arguments of up to 1.5 max|s| + 32: 2^-22 (1.5 max|s| + 32). The sums of
    weights and products over the blocks: 2^-23 per block and 64 beside. The weights of the second product are rounded
    to 2^-11 (F16) or 2^-21 (F32), and never below 2^-30 of the largest contribution per row. F16 outputs are rounded
    once more, 2^-11."""
    N, n, heads, d = q.shape
    g = heads // ref.H
    off, rel = np.zeros(q.shape), np.zeros((N, ref.H))
    for i in range(N):
        s = seq0 + i
        L = ref.len(s)
        for h in range(ref.H):
            k, v, bad = ref.rows(s, h)
            k, v = np.where(bad[:, None], 0, k), np.where(bad[:, None], 0, v)
            for j in range(n):
                m = L - n + 1 + j
                if m <= 0:
                    continue
                for a in range(h * g, h * g + g):
                    x = q[i, j, a].astype(np.float64)
                    mag = abs(scale) * (np.abs(k[:m]) @ np.abs(x)).max()
                    sc = scale * (k[:m] @ x)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    e = 2 * mag * ((d + 8) * 2.0 ** -23 + 2.0 ** -22) + (1.5 * np.abs(sc).max() + 32) * 2.0 ** -22 + \
                        (64 + 4 * -(-m // B)) * 2.0 ** -23
                    rel[i, h] = max(rel[i, h], e)
                    r = e + (2.0 ** -11 if f16 else 2.0 ** -21)
                    off[i, j, a] = r * (p @ np.abs(v[:m])) + m * 2.0 ** -30 * np.abs(v[:m]).max()
                    if f16:
                        off[i, j, a] += 2.0 ** -11 * np.abs(p @ v[:m]) + 2.0 ** -24
    return off, rel


def check_attend(dev, ref, q, scale, dtype=moert.F32, decay=None, seq0=0):
    if dtype == moert.F16:
        q = q.astype(np.float16)
    before = [[[b[4] for b in ref.blocks[s][h]] + [ref.tail_mass[s, h]] for h in range(ref.H)] for s in range(ref.S)]
    want = ref.attend(q, scale, decay, seq0)
    got = dev.attend(q, scale, dtype, decay, seq0=seq0).astype(np.float64)
    off, rel = out_bound(ref, q, scale, dtype == moert.F16, seq0)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    worst = np.abs(got - want)[fine] / np.maximum(off[fine], 1e-300)
    assert (np.abs(got - want)[fine] <= off[fine]).all(), f"out: {worst.max()} of its bound"
    if decay is not None:
        for i in range(q.shape[0]):
            s = seq0 + i
            nb = -(-ref.len(s) // B)
            for h in range(ref.H):
                have = dev.mass(s, h, nb).astype(np.float64)
                full = len(ref.blocks[s][h])
                need = np.array([b[4] for b in ref.blocks[s][h]] + [ref.tail_mass[s, h]] * (nb - full))
                assert np.array_equal(np.isnan(have), np.isnan(need)), (s, h)
                old = np.array(before[s][h][:full] + [before[s][h][-1]] * (nb - full))
                w = need - decay * old
                # the weights' bound; each of the n x group additions and the last fma round what is there already
                lim = rel[i, h] * w + need * (q.shape[1] * q.shape[2] / ref.H + 4) * 2.0 ** -23
                ok = ~np.isnan(need)
                assert (np.abs(have - need)[ok] <= lim[ok] + 1e-37).all(), (s, h, np.abs(have - need), lim)
                # from here on both go on from the same masses
                for b, blk in enumerate(ref.blocks[s][h]):
                    blk[4] = have[b]
                if nb > full:
                    ref.tail_mass[s, h] = have[-1]
    return got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_appends_hold_what_the_definition_says(hip, d, dtype):
    dev, ref = both(hip, 3, 3, d, 512)
    rng = np.random.default_rng(d + dtype)
    for n, seq0, count in ((1, 0, 3), (1, 1, 2), (30, 0, 1), (1, 0, 1), (1, 0, 1), (31, 1, 1), (32, 2, 1), (33, 0, 3),
                           (1, 0, 3), (64, 1, 2), (95, 0, 1), (127, 0, 2), (2, 0, 3)):
        print(f"[case] append {n} rows to sequences {seq0} + {count}", flush=True)
        k, v = normal(rng, count, n, 3, d), normal(rng, count, n, 3, d, scale=3.0)
        k[0, 0] *= 100.0
        dev.append(k, v, dtype, seq0=seq0)
        ref.append(k, v, seq0)
        ku.assert_holds(dev, ref)
    assert dev.c.lengths().tolist() == [ref.len(s) for s in range(3)]


def test_codes_at_ties_and_extremes(hip):
    """Ties of the quotient, subnormal fp16 rows, the largest fp16, zero blocks."""
    dev, ref = both(hip, 1, 2, 64, 256)
    rows = np.zeros((1, 192, 2, 64), np.float32)
    rng = np.random.default_rng(3)
    rows[0, :32, 0] = rng.integers(-254, 255, (32, 64)) / 2.0  # scale 1: every half is a tie
    rows[0, 0, 0, 0] = 127.0
    rows[0, 32:64, 0] = rng.integers(-8, 9, (32, 64)) * 2.0 ** -24
    rows[0, 64:96, 0] = rng.uniform(-65504, 65504, (32, 64))
    rows[0, 96:128, 0] = rng.integers(-254, 255, (32, 64)) * 2.0 ** -16
    rows[0, 128:160, 0] = rng.standard_normal((32, 64)) * 1e-6
    rows[0, 160:, 1] = rng.integers(-127, 128, (32, 64)) * 0.0625
    back = rows[:, :, ::-1]
    dev.append(rows, back)
    ref.append(rows, back)
    ku.assert_holds(dev, ref)


@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_strided_rows(hip, dtype):
    """K and V out of one product's rows [position][q | k | v], and out of a cache [head][position][element]; queries and
    outputs between other data, which stays."""
    t = np.float32 if dtype == moert.F32 else np.float16
    rng = np.random.default_rng(8)
    S, H, g, d, n = 2, 2, 3, 64, 37
    dev, ref = both(hip, S, H, d, 128)
    wide = (g * H + 2 * H) * d + 5
    qkv = normal(rng, S, n, wide).astype(t)
    at = hip.upload(qkv)
    size = qkv.itemsize
    st = (n * wide, wide, d)
    dev.c.append(at + (g * H * d + 1) * size, at + ((g * H + H) * d + 3) * size, n, dtype=dtype, strides=st)
    k = qkv[:, :, g * H * d + 1:][:, :, :H * d].reshape(S, n, H, d)
    v = qkv[:, :, (g * H + H) * d + 3:][:, :, :H * d].reshape(S, n, H, d)
    ref.append(k, v)
    ku.assert_holds(dev, ref)
    planes = normal(rng, S, H, n, d).astype(t)  # as moert_read_kv_fp16 gives them
    at2 = hip.upload(planes)
    dev.c.append(at2, at2, n, dtype=dtype, strides=(H * n * d, d, n * d))
    ref.append(planes.transpose(0, 2, 1, 3), planes.transpose(0, 2, 1, 3))
    ku.assert_holds(dev, ref)
    # attention of the last 5 positions, q inside the first product's rows, out with a gap of 7 after each head
    m = 5
    q = qkv[:, -m:, :g * H * d].reshape(S, m, g * H, d)
    out = np.full((S, m, g * H, d + 7), 9.0, t)
    out_at = hip.upload(out)
    ws, bytes_ = dev.workspace(g * H, m, S, False)
    dev.c.attend(at + (n - m) * wide * size, out_at, g * H, m, 0.125, ws, bytes_, dtype=dtype, q_strides=st,
                 out_strides=(m * g * H * (d + 7), g * H * (d + 7), d + 7))
    hip.sync()
    got = hip.get(out_at, out.shape, t)
    assert (got[..., d:] == 9.0).all()
    off, _ = out_bound(ref, q, 0.125, dtype == moert.F16)
    assert (np.abs(got[..., :d].astype(np.float64) - ref.attend(q, 0.125)) <= off).all()


SHAPES = [(1, 1, 64), (8, 2, 64), (8, 3, 64), (2, 4, 128), (4, 8, 64), (1, 6, 128), (2, 17, 64), (1, 64, 64)]


@pytest.mark.parametrize("kv_heads,group,d", SHAPES)
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_single_tokens_at_every_kind_of_length(hip, kv_heads, group, d, dtype):
    """One position after 0, 1, .. rows: tails, block ends, several splits."""
    lens = [1, 2, 31, 32, 33, 63, 64, 65, 130, 257, 511]
    S = len(lens)
    dev, ref = both(hip, S, kv_heads, d, 544)
    rng = np.random.default_rng(kv_heads * 100 + group)
    for s, n in enumerate(lens):
        k, v = normal(rng, 1, n, kv_heads, d), normal(rng, 1, n, kv_heads, d, scale=2.0)
        dev.append(k, v, seq0=s)
        ref.append(k, v, s)
    print(f"[case] heads {kv_heads} x {group} of {d}", flush=True)
    q = normal(rng, S, 1, kv_heads * group, d, scale=2.0)
    check_attend(dev, ref, q, d ** -0.5, dtype)
    check_attend(dev, ref, q, d ** -0.5, dtype, decay=1.0)
    check_attend(dev, ref, normal(rng, *q.shape, scale=4.0), -0.5 * d ** -0.5, dtype, decay=0.25)


@pytest.mark.parametrize("kv_heads,group,d,dtype,length,n", [
    (8, 3, 64, moert.F32, 70, 5), (8, 3, 64, moert.F16, 300, 33), (2, 2, 128, moert.F32, 100, 64),
    (1, 4, 64, moert.F16, 257, 257), (2, 3, 64, moert.F32, 333, 130), (1, 8, 128, moert.F16, 96, 96),
    (2, 1, 64, moert.F32, 65, 2), (1, 1, 64, moert.F16, 40, 31)])
def test_several_positions_see_their_own_rows(hip, kv_heads, group, d, dtype, length, n):
    """A ragged batch of two sequences, whose positions each see their row and those before; then the next part."""
    dev, ref = both(hip, 2, kv_heads, d, 512)
    rng = np.random.default_rng(length * 7 + n)
    for s, m in ((0, length), (1, max(n, length // 2))):
        k, v = normal(rng, 1, m, kv_heads, d), normal(rng, 1, m, kv_heads, d)
        dev.append(k, v, seq0=s)
        ref.append(k, v, s)
    print(f"[case] {n} positions of {length}, heads {kv_heads} x {group} of {d}", flush=True)
    q = normal(rng, 2, n, kv_heads * group, d, scale=2.0)
    check_attend(dev, ref, q, d ** -0.5, dtype)
    check_attend(dev, ref, q, d ** -0.5, dtype, decay=1.0)
    k, v = normal(rng, 2, 17, kv_heads, d), normal(rng, 2, 17, kv_heads, d)
    dev.append(k, v, dtype)
    ref.append(k if dtype == moert.F32 else k.astype(np.float16), v, 0)
    check_attend(dev, ref, normal(rng, 2, 17, kv_heads * group, d), d ** -0.5, dtype, decay=0.5)


@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_positions_that_see_nothing_get_zero(hip, dtype):
    """More positions than rows, a sequence of no rows, and the masses of what is seen all the same."""
    dev, ref = both(hip, 3, 2, 64, 128)
    rng = np.random.default_rng(4)
    for s, m in ((0, 3), (1, 40)):
        k, v = normal(rng, 1, m, 2, 64), normal(rng, 1, m, 2, 64)
        dev.append(k, v, seq0=s)
        ref.append(k, v, s)
    got = check_attend(dev, ref, normal(rng, 3, 48, 4, 64), 0.125, dtype, decay=1.0)
    assert not got[0, :45].any() and got[0, 45:].all() and not got[1, :8].any() and not got[2].any()


@pytest.mark.parametrize("n", [1, 20])
def test_long_contexts_in_many_splits(hip, n):
    dev, ref = both(hip, 1, 2, 64, 16384)
    rng = np.random.default_rng(6)
    k, v = normal(rng, 1, 9001, 2, 64), normal(rng, 1, 9001, 2, 64)
    dev.append(k, v)
    ref.append(k, v)
    for dtype in (moert.F32, moert.F16):
        check_attend(dev, ref, normal(rng, 1, n, 6, 64, scale=3.0), 0.125, dtype, decay=1.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_one_long_sequence_among_many(hip, d, dtype):
    """128 sequences, most of a few rows or none, one of 9001: no splits, and more blocks to a wave than one of its
    rounds of 64 holds."""
    S, H, g = 128, 8, 2
    dev, ref = ku.Device(hip, S, H, d, 9216, fill=False), ku.Cache(S, H, d, 9216)
    rng = np.random.default_rng(21)
    for s, m in ((5, 9001), (0, 1), (17, 33), (64, 64), (127, 300)):
        k, v = normal(rng, 1, m, H, d), normal(rng, 1, m, H, d)
        dev.append(k, v, seq0=s)
        ref.append(k, v, s)
    q = normal(rng, S, 1, H * g, d, scale=2.0)
    got = check_attend(dev, ref, q, d ** -0.5, dtype, decay=1.0)
    assert not got[[1, 2, 100]].any()
    got = check_attend(dev, ref, q, d ** -0.5, dtype)
    assert got[5].all()


def test_offsets_beyond_32_bits(hip):
    """Five sequences of 2^20 positions and 1 GiB of K codes each, the last one's blocks in its last slots."""
    S, H, d, max_len = 5, 8, 128, 1 << 20
    dev, ref = ku.Device(hip, S, H, d, max_len, fill=False), ku.Cache(S, H, d, max_len)
    table = dev.array("table")
    dev.set("table", table[:, :, ::-1].copy())
    rng = np.random.default_rng(22)
    for m in (150, 1, 60, 200):
        k, v = normal(rng, 1, m, H, d), normal(rng, 1, m, H, d)
        dev.append(k, v, seq0=4)
        ref.append(k, v, 4)
        for dtype in (moert.F32, moert.F16):
            check_attend(dev, ref, normal(rng, 1, 1, H * 2, d), 0.1, dtype, decay=1.0, seq0=4)
    check_attend(dev, ref, normal(rng, 1, 5, H * 8, d), 0.1, moert.F16, decay=1.0, seq0=4)
    dev.c.evict(6, first=1, last=1, seq0=4)
    ref.evict(6, 1, 1, 4, 1)
    assert dev.c.lengths().tolist() == [0, 0, 0, 0, 6 * 32 + 411 % 32]
    check_attend(dev, ref, normal(rng, 1, 3, H * 2, d), 0.1, decay=1.0, seq0=4)
    k, v = normal(rng, 1, 40, H, d), normal(rng, 1, 40, H, d)
    dev.append(k, v, seq0=4)
    ref.append(k, v, 4)
    shape = (1, 240, H, d)
    at = [hip.alloc(int(np.prod(shape)) * 4) for _ in range(2)]
    dev.c.read(at[0], at[1], 0, 240, seq0=4, n_seqs=1)
    hip.sync()
    for x, want in zip(at, ref.read(4, 0, 240)):
        assert np.array_equal(hip.get(x, shape, np.float32)[0], want.astype(np.float32))


def test_a_scale_of_zero_weighs_every_row_alike(hip):
    dev, ref = both(hip, 1, 2, 64, 256)
    rng = np.random.default_rng(23)
    r = normal(rng, 2, 1, 203, 2, 64)
    dev.append(r[0], r[1])
    ref.append(r[0], r[1])
    for n in (1, 40):
        for dtype in (moert.F32, moert.F16):
            check_attend(dev, ref, normal(rng, 1, n, 4, 64), 0.0, dtype, decay=1.0)


def test_scales_far_apart(hip):
    """Blocks of V whose scales differ by 2^30, with the attention on the small ones: sums keep what the type holds.
    Queries from 2^-60 to 2^60 beside keys that make ordinary scores."""
    dev, ref = both(hip, 1, 1, 64, 512)
    rng = np.random.default_rng(9)
    k, v = normal(rng, 1, 300, 1, 64), normal(rng, 1, 300, 1, 64)
    for b in range(10):
        v[:, b * 32:b * 32 + 32] *= 2.0 ** (-14 + 3 * b if b % 2 else -14)
        k[:, b * 32:b * 32 + 32] *= 2.0 ** (-b)
    dev.append(k, v)
    ref.append(k, v)
    q = normal(rng, 1, 1, 4, 64)
    q *= np.array([2.0 ** -60, 1.0, 2.0 ** 60, 3.0], np.float32)[:, None]
    q[:, :, 2, :-1] = 0.0  # one product a score: 2^60 k, whose differences leave one row
    check_attend(dev, ref, q, 1.0)
    check_attend(dev, ref, q * 2.0 ** 60, 2.0 ** -60)


@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_poison_reaches_what_sees_it_and_nothing_else(hip, dtype):
    """inf, NaN and an f32 beyond fp16, in a coded block, in the tail, in rows behind the sequence."""
    for name, row in (("block", 40), ("tail", 97), ("tail end", 99)):
        for kv in (0, 1):
            for value in (np.inf, -np.inf, np.nan, 1e6):
                print(f"[case] {value} in {'kv'[kv]}, {name}", flush=True)
                dev, ref = both(hip, 1, 2, 64, 128)
                rng = np.random.default_rng(11)
                r = normal(rng, 2, 1, 100, 2, 64)
                r[kv, 0, row, 1, 7] = value
                dev.append(r[0], r[1])
                ref.append(r[0], r[1])
                ku.assert_holds(dev, ref)
                got = check_attend(dev, ref, normal(rng, 1, 70, 4, 64), 0.125, dtype, decay=1.0)
                assert not np.isnan(got[:, :, :2]).any() and np.isnan(got[:, -1, 2:]).all()
                k, v = dev.read(0, 100)
                wk, wv = ref.read(0, 0, 100)
                assert np.array_equal(np.isnan(k[0]), np.isnan(wk)) and np.array_equal(np.isnan(v[0]), np.isnan(wv))


@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_queries_that_are_not_finite(hip, dtype):
    """NaN and inf in one query head's row: that row is NaN, the others are what they were; also where every score is
    -inf, of one row and of many, with and without splits."""
    rng = np.random.default_rng(12)
    for length, max_len in ((77, 128), (1, 128), (64, 128), (1000, 16384)):
        dev = ku.Device(hip, 1, 2, 64, max_len)
        r = normal(rng, 2, 1, length, 2, 64)
        r[0, :, :, :, 5] = -np.abs(r[0, :, :, :, 5]) - 1.0
        dev.append(r[0], r[1])
        for n in (1, 3):
            q = normal(rng, 1, n, 6, 64)
            want = dev.attend(q, 0.125, dtype)
            bad = q.copy()
            bad[0, 0, 2, 5], bad[0, n - 1, 4, 5], bad[0, n - 1, 1, 0] = np.nan, np.inf, -np.inf
            got = dev.attend(bad, 0.125, dtype)
            hit = np.zeros((1, n, 6), bool)
            hit[0, 0, 2] = hit[0, n - 1, 4] = hit[0, n - 1, 1] = True
            seen = np.broadcast_to((length - n + 1 + np.arange(n) > 0)[None, :, None], hit.shape)
            assert np.isnan(got[hit & seen]).all() and not got[hit & ~seen].any(), (length, n)
            assert np.array_equal(got[~hit], want[~hit]), (length, n)


def test_scores_beyond_f32_are_not_zero_outputs(hip):
    """Every score -1e42: NaN, as f32 softmax has it, not the 0 of a position that sees nothing."""
    dev = ku.Device(hip, 1, 1, 64, 128)
    k = np.full((1, 40, 1, 64), -1e4, np.float32)
    dev.append(k, k)
    q = np.full((1, 2, 1, 64), 1e37, np.float32)
    assert np.isnan(dev.attend(q, 1.0)).all()
    dev.attend(q, 1.0, decay=1.0)
    assert np.isnan(dev.mass(0, 0, 2)).all()


@pytest.mark.parametrize("decay", [None, 0.5])
@pytest.mark.parametrize("max_len", [384, 8192])
def test_the_largest_values_stay_finite(hip, max_len, decay):
    """V of fp16's largest magnitude and, in all rows that count, weights whose rounding to fp16 has one sign: 64 heads
    whose scores lie 1 .. 7.3 (in base 2) above the rows that set each wave's maximum. An output is off by half a step
    of its weights at most, and the exact one, +-65504, is the type's last number: nothing becomes infinite."""
    d, rows = 64, 384
    dev, ref = both(hip, 1, 1, d, max_len)
    k, v = np.zeros((1, rows, 1, d)), np.full((1, rows, 1, d), 65504.0)
    k[:, rows // 2:, :, 0] = 1.0  # the first blocks, every wave's first, score 0
    v[..., 1::2] = -65504.0
    dev.append(k, v)
    ref.append(k, v)
    q = np.zeros((1, 1, 64, d))
    q[..., 0] = 0.7 + np.arange(64) / 14.5
    out = check_attend(dev, ref, q.astype(np.float16), 1.0, dtype=moert.F16, decay=decay)
    assert np.isfinite(out).all()


@pytest.mark.parametrize("n", [1, 9])
def test_scores_near_f32s_lowest(hip, n):
    """Scores of about -1e36, apart by 1e34 and more: all the weight is on the least negative one that is seen."""
    rng = np.random.default_rng(23)
    d, rows = 64, 700
    dev, ref = both(hip, 1, 2, d, 1024)
    k, v = np.zeros((1, rows, 2, d)), normal(rng, 1, rows, 2, d)
    k[..., 0] = 127.0  # of a scale of 1 in every block
    for h in range(2):
        k[0, 40 + 300 * h, h, 0] = 100.0
    dev.append(k, v)
    ref.append(k, v)
    q = np.zeros((1, n, 4, d), np.float32)
    q[..., 0] = -1e34
    out = dev.attend(q, 1.0, decay=0.0)
    for h in range(2):
        want = ref.rows(0, h)[1][40 + 300 * h]
        for a in (2 * h, 2 * h + 1):
            # weights of one row, a code and a scale: three roundings of 2^-24
            assert np.abs(out[0, :, a] - want).max() <= 4 * 2.0 ** -24 * np.abs(want).max()
        mass = dev.mass(0, h, -(-rows // 32))
        assert mass[(40 + 300 * h) // 32] == 2 * n and mass.sum() == 2 * n


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_reads(hip, d, dtype):
    dev, ref = both(hip, 2, 3, d, 256)
    rng = np.random.default_rng(13)
    for s, m in ((0, 150), (1, 64)):
        r = normal(rng, 2, 1, m, 3, d)
        dev.append(r[0], r[1], seq0=s)
        ref.append(r[0], r[1], s)
    t = np.float32 if dtype == moert.F32 else np.float16
    for pos, n in ((0, 1), (0, 256), (31, 2), (100, 70), (-1, 1), (-64, 64), (-150, 33), (-256, 256), (255, 256)):
        print(f"[case] read {n} from {pos}", flush=True)
        k, v = dev.read(pos, n, dtype)
        for s in range(2):
            for got, want in zip((k, v), ref.read(s, pos, n)):
                assert np.array_equal(got[s], want.astype(np.float32).astype(t)), (s, pos, n)


def test_appends_without_room_leave_the_sequence(hip):
    dev, ref = both(hip, 2, 2, 64, 64)
    rng = np.random.default_rng(14)
    r = normal(rng, 2, 1, 60, 2, 64)
    dev.append(r[0], r[1], seq0=1)
    ref.append(r[0], r[1], 1)
    for n in (5, 1, 1, 2, 64):
        r = normal(rng, 2, 2, n, 2, 64)
        dev.append(r[0], r[1])
        ref.append(r[0], r[1])
        ku.assert_holds(dev, ref)
    assert ref.dropped == [64, 5 + 64]
    with pytest.raises(moert.MoertError) as e:
        dev.c.lengths()
    assert e.value.code == moert.E_FULL and "sequence 0" in str(e.value)
    dev.c.clear(seq0=0, n_seqs=1)
    assert dev.c.lengths(0, 1).tolist() == [0]
    with pytest.raises(moert.MoertError):
        dev.c.lengths(1, 1)


def test_lengths_come_with_the_report_of_dropped_rows(hip):
    dev, _ = both(hip, 3, 1, 64, 64)
    x = np.ones((1, 40, 1, 64))
    dev.append(x, x, seq0=1)
    dev.append(x, x, seq0=1)
    dev.append(x[:, :7], x[:, :7], seq0=2)
    with pytest.raises(moert.MoertError) as e:
        dev.c.lengths()
    assert e.value.code == moert.E_FULL and e.value.lengths.tolist() == [0, 40, 7]


def set_masses(dev, ref, masses):
    """masses(s, h, blocks) -> f32 of every block in use, set on both sides."""
    m = dev.array("mass")
    table = dev.array("table")
    for s in range(ref.S):
        for h in range(ref.H):
            nb, full = -(-ref.len(s) // B), len(ref.blocks[s][h])
            x = masses(s, h, nb).astype(np.float32)
            m[s, h, table[s, h, :nb]] = x
            for b in range(full):
                ref.blocks[s][h][b][4] = x[b]
            if nb > full:
                ref.tail_mass[s, h] = x[-1]
    dev.set("mass", m)


@pytest.mark.parametrize("max_len,lens", [(320, (7, 64, 300)), (16384, (8256, 8191, 8259)), (2 ** 15, (30000,)),
                                          (65536, (40000, 33000)), (2 ** 17, (130001,)), (2 ** 18, (2 ** 18 - 5,)),
                                          (2 ** 20, (2 ** 20 - 3,))])
def test_evictions(hip, max_len, lens):
    """Masses with ties, zeros, infinities and NaN; budgets from 0 to more than there is; what stays is as it was."""
    S = len(lens)
    few = max_len <= 320
    H = 3 if few else 1
    rng = np.random.default_rng(15)
    for keep, first, last in ((0, 0, 0), (1, 0, 0), (1, 1, 0), (1, 0, 1), (3, 1, 1), (2, 1, 1), (5, 0, 2), (4, 2, 1),
                              (9, 0, 0), (500, 1, 4)):
        if not few:
            keep, first, last = keep * 113, first * 5, last * 7
        for kind in ("spread", "equal", "odd"):
            print(f"[case] lengths {lens}, keep {keep}, first {first}, last {last}, {kind}", flush=True)
            dev, ref = ku.Device(hip, S, H, 64, max_len, fill=few), ku.Cache(S, H, 64, max_len)
            for s, n in enumerate(lens):
                r = normal(rng, 2, 1, n if few else 64 + n % 32, H, 64)
                dev.append(r[0], r[1], seq0=s)
                ref.append(r[0], r[1], s)
                if not few:  # the length alone counts
                    st = dev.array("state")
                    st[s, 0] = n
                    dev.set("state", st)
                    ref.blocks[s][0] = [[None, None, None, None, 0.0] for _ in range(n // B)]
            order = np.stack([np.stack([rng.permutation(max_len // B) for _ in range(H)]) for _ in range(S)])
            if few:
                order = dev.array("table")  # blocks have been written to their slots
            dev.set("table", order)

            def masses(s, h, nb):
                if kind == "spread":
                    return np.exp(2 * rng.standard_normal(nb))
                x = rng.choice([0.0, 1.0, 1.0, 2.5], nb)
                if kind == "odd":
                    x = np.where(rng.random(nb) < 0.2, rng.choice([np.inf, np.nan, -0.0, 1e-40, 3e38], nb), x)
                return x

            set_masses(dev, ref, masses)
            table0, mass0 = dev.array("table"), dev.array("mass")
            where = [[{id(x): b for b, x in enumerate(ref.blocks[s][h])} for h in range(H)] for s in range(S)]
            full0 = [len(ref.blocks[s][0]) for s in range(S)]
            ref.evict(keep, first, last)
            dev.c.evict(keep, first=first, last=last)
            table, mass, state = dev.array("table"), dev.array("mass"), dev.array("state")
            for s in range(S):
                r = lens[s] % B
                assert state[s].tolist() == [len(ref.blocks[s][0]) * B + r, 0, 0, 0]
                for h in range(H):
                    stay = [where[s][h][id(x)] for x in ref.blocks[s][h]]
                    tail = [full0[s]] if r else []
                    kept = set(stay)
                    gone = [b for b in range(full0[s]) if b not in kept]
                    rest = list(range(full0[s] + len(tail), max_len // B))
                    assert table[s, h].tolist() == table0[s, h][stay + tail + gone + rest].tolist(), (s, h)
                    want = mass0[s, h].copy()
                    want[table0[s, h][gone]] = 0.0
                    assert np.array_equal(mass[s, h].view(np.uint32), want.view(np.uint32)), (s, h)


def test_evicted_caches_go_on(hip):
    """A run of the operators as a program has them: rows come, attention keeps the weights, evictions take the blocks
    that got least, more rows come into the slots that are free; every step against the definition."""
    rng = np.random.default_rng(16)
    dev, ref = both(hip, 2, 2, 64, 256)
    for step in range(24):
        n = [1, 40, 1, 7, 33, 1][step % 6]
        r = normal(rng, 2, 2, n, 2, 64)
        dtype = moert.F16 if step % 4 == 3 else moert.F32
        dev.append(r[0], r[1], dtype)
        ref.append(r[0].astype(np.float16), r[1].astype(np.float16))
        check_attend(dev, ref, normal(rng, 2, n, 6, 64, scale=2.0), 0.125, dtype, decay=0.9)
        if ref.len(0) > 170:
            print(f"[case] step {step}: eviction at {ref.len(0)}", flush=True)
            dev.c.evict(3, first=1, last=1)
            ref.evict(3, 1, 1)
            ku.assert_holds(dev, ref)
            check_attend(dev, ref, normal(rng, 2, 2, 6, 64), 0.125, decay=1.0)
    ku.assert_holds(dev, ref)


def test_a_captured_step_replays_from_the_lengths_it_finds(hip):
    """Append, attention with masses and eviction in one graph, replayed with eager work and synchronisations between,
    against the same calls made one by one on another cache."""
    rng = np.random.default_rng(17)
    S, H, g, d, max_len = 2, 2, 3, 64, 256
    one, two = (ku.Device(hip, S, H, d, max_len) for _ in range(2))
    stream = hip.stream()
    n_max = 60
    r = normal(rng, 2, S, 50, H, d)
    for dev in (one, two):
        dev.append(r[0], r[1])
    k, v, q = (hip.alloc(S * x * d * 4) for x in (H, H, H * g))
    outs = [hip.alloc(S * H * g * d * 4) for _ in range(2)]

    def step(dev, out, s):
        dev.c.append(k, v, 1, stream=s)
        ws, size = dev.workspace(H * g, 1, S, True)
        dev.c.attend(q, out, H * g, 1, 0.125, ws, size, mass_decay=1.0, stream=s)
        dev.c.evict(2, first=1, stream=s)

    one.workspace(H * g, 1, S, True)
    hip.sync()
    graph = hip.capture(stream, lambda: step(one, outs[0], stream))
    assert one.c.lengths(stream=stream).tolist() == [50, 50]  # a capture does nothing
    for i in range(n_max):
        hip.put(k, normal(rng, S, 1, H, d))
        hip.put(v, normal(rng, S, 1, H, d))
        hip.put(q, normal(rng, S, 1, H * g, d))
        hip.launch(graph, stream)
        step(two, outs[1], 0)
        hip.sync()
        a, b = (hip.get(o, (S, H * g, d), np.float32) for o in outs)
        assert np.array_equal(a, b), i
    for name in one.shapes:
        if name not in ("k_tail", "v_tail", "tail_bad", "k_codes", "v_codes", "k_scale", "v_scale"):
            assert np.array_equal(one.array(name), two.array(name)), name
    with pytest.raises(moert.MoertError) as e:
        hip.capture(stream, lambda: one.c.lengths(stream=stream))
    assert e.value.code == moert.E_CONFIG


def test_two_graphs_of_one_cache_and_workspace(hip):
    """A graph that appends and attends with five positions and one that only attends with masses, sharing the
    workspace, replayed in turn on one stream; against the same calls made one by one."""
    rng = np.random.default_rng(20)
    S, H, g, d, max_len, n = 2, 2, 4, 64, 512, 5
    one, two = (ku.Device(hip, S, H, d, max_len) for _ in range(2))
    stream = hip.stream()
    k, v, q = (hip.alloc(S * n * x * d * 2) for x in (H, H, H * g))
    size = one.c.workspace(H * g, n, track=True)
    ws = hip.alloc(size)
    outs = [[hip.alloc(S * n * H * g * d * 2) for _ in range(2)] for _ in range(2)]

    def chunk(dev, o, s):
        dev.c.append(k, v, n, dtype=moert.F16, stream=s)
        dev.c.attend(q, o[0], H * g, n, 0.125, ws, size, dtype=moert.F16, stream=s)

    def last(dev, o, s):
        dev.c.attend(q, o[1], H * g, 1, 0.125, ws, size, dtype=moert.F16, mass_decay=0.5, stream=s)

    hip.sync()
    graphs = [hip.capture(stream, lambda: f(one, outs[0], stream)) for f in (chunk, last)]
    for i in range(30):
        for at, heads in ((k, H), (v, H), (q, H * g)):
            hip.put(at, normal(rng, S, n, heads, d).astype(np.float16))
        for graph in graphs:
            hip.launch(graph, stream)
        hip.sync()
        chunk(two, outs[1], 0)
        last(two, outs[1], 0)
        hip.sync()
        for j, m in ((0, n), (1, 1)):
            a, b = (hip.get(o[j], (S, m, H * g, d), np.float16) for o in outs)
            assert np.array_equal(a, b) and a.any(), (i, j)
    assert np.array_equal(one.array("mass"), two.array("mass"))
    assert one.c.lengths().tolist() == [150, 150]


def test_attentions_on_two_streams(hip):
    """Attentions that do not track may overlap, each with a workspace of its own; results do not depend on it."""
    rng = np.random.default_rng(18)
    dev, ref = both(hip, 1, 2, 64, 4096)
    r = normal(rng, 2, 1, 3001, 2, 64)
    dev.append(r[0], r[1])
    q = normal(rng, 8, 1, 1, 8, 64)
    want = [dev.attend(x, 0.125) for x in q]
    size = dev.c.workspace(8, 1)
    streams = [hip.stream(), hip.stream()]
    ws = [hip.alloc(size) for _ in streams]
    qs, outs = [hip.upload(x) for x in q], [hip.alloc(8 * 64 * 4) for _ in q]
    hip.sync()
    for _ in range(3):
        for i in range(8):
            dev.c.attend(qs[i], outs[i], 8, 1, 0.125, ws[i % 2], size, stream=streams[i % 2])
        hip.sync()
        for i in range(8):
            assert np.array_equal(hip.get(outs[i], (1, 1, 8, 64), np.float32), want[i]), i


def test_a_broken_table_stays_inside_the_buffers(hip):
    """Entries outside the slots are taken as slot 0: values are of no use, memory is not touched outside."""
    dev, ref = both(hip, 1, 2, 64, 128)
    rng = np.random.default_rng(19)
    r = normal(rng, 2, 1, 100, 2, 64)
    dev.append(r[0], r[1])
    zero = dev.array("table")
    zero[:] = 0
    dev.set("table", zero)
    q = normal(rng, 1, 2, 4, 64)
    want, read = dev.attend(q, 0.125), dev.read(0, 96)
    dev.set("table", np.array([[[-1, 4, 2 ** 31 - 1, -2 ** 31]] * 2], np.int32))
    assert np.array_equal(dev.attend(q, 0.125), want)
    got = dev.read(0, 96)
    assert np.array_equal(got[0], read[0]) and np.array_equal(got[1], read[1])
    for length in (-5, 2 ** 30):
        st = dev.array("state")
        st[0, 0] = length
        dev.set("state", st)
        got = dev.attend(q, 0.125, decay=1.0)
        assert np.isfinite(got).all() and got.any() == (length > 0)
        dev.c.evict(1)


def weights_bound(ref, q, scale, f16):
    """How far an output may be from the 64-bit one, element by element, whatever the scales of V: e, the relative error
    of a weight in f32, is out_bound's. The weights of the second product are rounded by 2^-11 (F16) or 2^-21 (F32) of
    themselves. Below that an fp16 has a step of 2^-24, an error of 2^-25, where the largest contribution to its column
    so far, weight x scale of V, is at 2^7 or above: 2^-32 of it, over the block's own scale; and where the scale of a
    block lies more than 2^8 below that of a contribution that set the maximum, its weights are taken relative to their
    own largest: 2^-32 of the largest weight. So an error never passes 2^-24 of the largest weight."""
    N, n, heads, d = q.shape
    g = heads // ref.H
    off = np.zeros(q.shape)
    for i in range(N):
        L = ref.len(i)
        for h in range(ref.H):
            k, v, _ = ref.rows(i, h)
            vs = np.repeat([np.float64(b[3]) for b in ref.blocks[i][h]] + [1.0], B)[:L]
            for j in range(n):
                m = L - n + 1 + j
                for a in range(h * g, h * g + g):
                    x = q[i, j, a].astype(np.float64)
                    mag = abs(scale) * (np.abs(k[:m]) @ np.abs(x)).max()
                    sc = scale * (k[:m] @ x)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    e = 2 * mag * ((d + 8) * 2.0 ** -23 + 2.0 ** -22) + (1.5 * np.abs(sc).max() + 32) * 2.0 ** -22 + \
                        (64 + 4 * -(-m // B)) * 2.0 ** -23
                    floor = np.minimum(2.0 ** -24 * p.max(), 2.0 ** -32 * (p * vs[:m]).max() / vs[:m])
                    floor = np.maximum(floor, 2.0 ** -32 * p.max())
                    off[i, j, a] = (e + (2.0 ** -11 if f16 else 2.0 ** -21)) * (p @ np.abs(v[:m])) + floor @ np.abs(v[:m])
                    if f16:
                        off[i, j, a] += 2.0 ** -11 * np.abs(p @ v[:m]) + 2.0 ** -24
    return off


def scaled_v(kind, rng, rows, kv_heads, d):
    """V whose blocks differ by scale, the large ones first."""
    v, b = normal(rng, 1, rows, kv_heads, d), np.arange(rows)[None, :, None, None] // B
    if kind == "falling":  # by 2^2 from block to block, 2^8 from one of a wave's to its next, 2^37 in all
        return v * 2.0 ** np.maximum(13.0 - 2 * b, -24.0)
    if kind == "large first":
        return v * np.where(b < 4, 1e4, 1e-6)
    if kind == "zeros first":
        return v * np.where(b < 5, 0.0, 1e-4)
    if kind == "zeros between":
        return v * np.where(b % 3 == 1, 0.0, 1e-2)
    assert kind == "by element"  # the first blocks hold element 0 alone, the others all but it
    e = np.arange(d) == 0
    return np.where(b < 4, np.where(e, 1e4, 0.0), np.where(e, 0.0, 1e-3)) * v


@pytest.mark.parametrize("kind", ["falling", "large first", "zeros first", "zeros between", "by element"])
@pytest.mark.parametrize("d,n", [(64, 1), (64, 30), (128, 1), (128, 30)])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_scales_of_v_that_fall(hip, dtype, d, n, kind):
    """A wave's blocks with ever smaller V, and blocks of zeros before others: every row keeps its share of the sum of
    softmax and of its block's weight, and outputs do not depend on whether the weights are kept."""
    rng = np.random.default_rng(24)
    rows = 500  # blocks 0, 4, 8, 12 are one wave's
    dev, ref = both(hip, 1, 2, d, 512)
    k, v = normal(rng, 1, rows, 2, d), scaled_v(kind, rng, rows, 2, d)
    dev.append(k, v)
    ref.append(k, v)
    for size in (0.5, 4.0):
        q = normal(rng, 1, n, 6, d, scale=size).astype(np.float16 if dtype == moert.F16 else np.float32)
        off = weights_bound(ref, q, d ** -0.5, dtype == moert.F16)
        want = ref.attend(q, d ** -0.5)
        plain = dev.attend(q, d ** -0.5, dtype)
        kept = check_attend(dev, ref, q, d ** -0.5, dtype, decay=1.0)
        for got in (plain, kept):
            worst = np.abs(got.astype(np.float64) - want) / off
            assert (worst <= 1).all(), f"{size}: {worst.max()} of its bound"
        same = np.array_equal(plain.astype(np.float64), kept)
        assert same, size


@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
@pytest.mark.parametrize("n", [1, 12])
def test_zero_rows_before_a_long_sequence(hip, dtype, n):
    """A padded prompt: 1000 rows of zeros in K and V, then small V, in many splits."""
    rng = np.random.default_rng(25)
    dev, ref = both(hip, 1, 2, 64, 16384)
    k, v = normal(rng, 1, 9001, 2, 64), normal(rng, 1, 9001, 2, 64, scale=1e-4)
    k[:, :1000], v[:, :1000] = 0.0, 0.0
    dev.append(k, v)
    ref.append(k, v)
    q = normal(rng, 1, n, 6, 64).astype(np.float16 if dtype == moert.F16 else np.float32)
    off, want = weights_bound(ref, q, 0.125, dtype == moert.F16), ref.attend(q, 0.125)
    for decay in (None, 1.0):
        got = check_attend(dev, ref, q, 0.125, dtype, decay=decay)
        worst = np.abs(got.astype(np.float64) - want) / off
        assert (worst <= 1).all(), f"{worst.max()} of its bound"


def test_an_error_the_caller_has_dealt_with_fails_no_call(hip):
    dev, ref = both(hip, 1, 2, 64, 128)
    rng = np.random.default_rng(26)
    r = normal(rng, 2, 1, 70, 2, 64)
    at = [hip.upload(x) for x in r]
    assert hip.rt.hipSetDevice(4096) != 0  # no such device: the thread's last error
    dev.c.append(at[0], at[1], 70)
    ref.append(r[0], r[1])
    ku.assert_holds(dev, ref)
    q = normal(rng, 1, 1, 4, 64)
    dev.workspace(4, 1, 1, True)
    assert hip.rt.hipSetDevice(4096) != 0
    check_attend(dev, ref, q, 0.125, decay=1.0)


@pytest.mark.parametrize("n", [40, 3000])
def test_dropped_rows_are_never_counted_back_to_none(hip, n):
    """Two appends without room, behind 2^31 - 100 dropped rows: the count stays at the largest number."""
    max_len = 32 * (n // 32 + 1)
    dev, _ = both(hip, 1, 8, 64, max_len)
    x = np.ones((1, n, 8, 64))
    dev.append(x, x)
    state = dev.array("state")
    state[0, 1] = 2 ** 31 - 100
    dev.set("state", state)
    for _ in range(2):
        dev.append(np.ones((1, max_len, 8, 64)), np.ones((1, max_len, 8, 64)))
    dev.append(x, x)
    assert dev.array("state")[0].tolist() == [n, 2 ** 31 - 1, 0, 0]
    with pytest.raises(moert.MoertError) as e:
        dev.c.lengths()
    assert e.value.code == moert.E_FULL and e.value.lengths.tolist() == [n]


@pytest.mark.parametrize("d,dtype", [(64, moert.F32), (128, moert.F16)])
def test_broken_tables_and_lengths_change_nothing_outside_the_buffers(hip, d, dtype):
    """The cache's arrays in one allocation with known bytes before, between and behind them; entries outside the slots
    and lengths outside the cache, met by every call that reads or writes through them."""
    S, H, max_len, guard = 2, 2, 256, 8192
    dev = ku.Device(hip, S, H, d, max_len)
    place, size = {}, guard
    for name, (shape, kind) in dev.shapes.items():
        place[name] = size
        size += -(-int(np.prod(shape)) * np.dtype(kind).itemsize // 16) * 16 + guard
    memory = np.full(size, 0xA5, np.uint8)
    base = hip.upload(memory)
    dev.at = {name: base + x for name, x in place.items()}
    dev.c = moert.Kv8(S, H, d, max_len, dev.at)
    dev.c.clear()
    outside = np.ones(size, bool)
    for name, (shape, kind) in dev.shapes.items():
        outside[place[name]:place[name] + int(np.prod(shape)) * np.dtype(kind).itemsize] = False
    rng = np.random.default_rng(27)
    slots = max_len // B
    broken = np.array([-1, slots, 2 ** 31 - 1, -2 ** 31, slots + 1, -2, 3, 2 ** 20], np.int64)
    for length in (0, 40, 200, -5, max_len + 1, 2 ** 30, 2 ** 31 - 1, -2 ** 31):
        print(f"[case] length {length}", flush=True)
        for rows in (1, 33, 128):
            state = np.zeros((S, 4), np.int32)
            state[:, 0] = length
            dev.set("state", state)
            dev.set("table", np.stack([np.stack([rng.permutation(broken) for _ in range(H)]) for _ in range(S)]))
            dev.append(normal(rng, S, rows, H, d), normal(rng, S, rows, H, d), dtype)
            for n in (1, 20):
                dev.attend(normal(rng, S, n, 3 * H, d), 0.125, dtype, decay=0.5)
            dev.read(-100, 256, dtype)
            dev.c.evict(1, first=1)
            dev.attend(normal(rng, S, 1, 3 * H, d), 0.125, dtype)
            hip.sync()
            now = hip.get(base, (size,), np.uint8)
            changed = np.flatnonzero(outside & (now != 0xA5))
            assert changed.size == 0, (length, rows, changed[:4])


@pytest.mark.parametrize("max_len", [256, 16384])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_outputs_in_place_of_the_queries(hip, dtype, max_len):
    """out = q, of the same strides: every row of q is read before its output is written, with and without splits."""
    rng = np.random.default_rng(28)
    t = np.float32 if dtype == moert.F32 else np.float16
    dev = ku.Device(hip, 2, 2, 64, max_len)
    r = normal(rng, 2, 2, max_len // 2 + 7, 2, 64)
    dev.append(r[0], r[1])
    for n in (1, 3, 70):
        q = normal(rng, 2, n, 6, 64).astype(t)
        for decay in (None, 1.0):
            want = dev.attend(q, 0.125, dtype, decay)
            at = hip.upload(q)
            ws, size = dev.workspace(6, n, 2, decay is not None)
            dev.c.attend(at, at, 6, n, 0.125, ws, size, dtype=dtype, mass_decay=decay)
            hip.sync()
            same = np.array_equal(hip.get(at, q.shape, t), want)
            assert same, (n, decay)


@pytest.mark.parametrize("d,heads,n", [(64, 16, 1), (64, 3, 5), (128, 8, 2), (128, 5, 1)])
@pytest.mark.parametrize("max_len", [1024, 16384])
def test_fp16_outputs_of_few_rows_are_off_by_their_own_rounding(hip, d, heads, n, max_len):
    """At most 16 query rows of a KV head: the weights keep 22 bits, as with f32, and the output is rounded once. All
    rows that count have one weight, so that roundings of weights would add up, whatever part of a step they take."""
    rng = np.random.default_rng(29)
    rows = 999
    dev, ref = both(hip, 1, 1, d, max_len)
    k, v = np.zeros((1, rows, 1, d)), np.broadcast_to(rng.uniform(1.0, 2.0, d), (1, rows, 1, d))
    k[:, rows // 2:, :, 0] = 1.0  # each wave's first block has score 0
    dev.append(k, v)
    ref.append(k, v)
    q = np.zeros((1, n, heads, d), np.float16)
    q[..., 0] = (0.7 + np.arange(n * heads) / 14.5).reshape(n, heads)
    want = ref.attend(q, 1.0)
    # half a step of the output: the steps of [1, 2) are 2^-10, those of [1/2, 1) half of that
    off = weights_bound(ref, q, 1.0, False) + np.where(np.abs(want) < 1.0, 2.0 ** -12, 2.0 ** -11)
    for decay in (None, 1.0):
        worst = np.abs(dev.attend(q, 1.0, moert.F16, decay).astype(np.float64) - want) / off
        assert (worst <= 1).all(), f"{worst.max()} of its bound"


def test_k_and_v_of_different_types(hip):
    """Each of the rows of a call has its own type and strides."""
    rng = np.random.default_rng(30)
    dev, ref = both(hip, 1, 2, 64, 128)
    k, v = normal(rng, 1, 77, 2, 64), normal(rng, 1, 77, 2, 64).astype(np.float16)
    lib, c = moert.lib(), dev.c
    rows = lambda at, dtype: c._rows(at, dtype, None, 77, 2)
    moert.check(lib.moert_kv8_append(c._p, 0, 1, rows(hip.upload(k), moert.F32), rows(hip.upload(v), moert.F16), 77, None))
    ref.append(k, v)
    ku.assert_holds(dev, ref)
    out = [hip.upload(np.full((77, 2, 64), 7.0, t)) for t in (np.float16, np.float32)]
    moert.check(lib.moert_kv8_read(c._p, 0, 1, 0, 77, rows(out[0], moert.F16), rows(out[1], moert.F32), None))
    hip.sync()
    for at, t, want in zip(out, (np.float16, np.float32), ref.read(0, 0, 77)):
        assert np.array_equal(hip.get(at, want.shape, t), want.astype(np.float32).astype(t))


@pytest.mark.parametrize("max_len,n", [(768, 1), (768, 20), (16384, 1), (16384, 12)])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_scores_of_any_size(hip, dtype, max_len, n):
    """Scores of 10^4 to 10^30, far beyond the steps of exponents: all the weight on one row, or shared by every 37th in
    equal parts, whatever the scales of V of their blocks."""
    rng = np.random.default_rng(31)
    d, rows = 64, 700
    b = np.arange(rows)[None, :, None, None] // B
    for kind, v_scale in (("ordinary", 1.0), ("small", 1e-3), ("rising", 2.0 ** (b % 7 * 3 - 10.0)), ("large", 1e4)):
        v = normal(rng, 1, rows, 2, d) * v_scale
        for every in (rows, 37):
            k = np.zeros((1, rows, 2, d), np.float32)
            k[..., 0], k[..., 1] = rng.integers(20, 100, (1, rows, 2)), 127.0  # a scale of 1 in every block
            k[0, 20::every, :, 0] = 127.0
            dev, ref = both(hip, 1, 2, d, max_len)
            dev.append(k, v)
            ref.append(k, v)
            at = np.arange(20, rows, every)
            for size in (1e4, 1e5, 1e6, 1e7, 3e7, 1e8, 3e8, 1e9, 4e9, 1e10, 1e12, 1e30):
                for sign in (1.0, -1.0):
                    q = np.zeros((1, n, 4, d), np.float32)
                    q[..., 0] = 16.0
                    if sign < 0:  # every score below 0, the same ones apart
                        q[..., 1] = -32.0
                    scale = size / (16.0 * 127.0)
                    for decay in (None, 0.0):
                        out = dev.attend(q.astype(np.float16) if dtype == moert.F16 else q, scale, dtype, decay)
                        for h in range(2):
                            x = ref.rows(0, h)[1]
                            for i in range(n):
                                w = at[at < rows - n + 1 + i]
                                want = x[w].mean(0)
                                # a weight: 22 bits or (F16, two tiles) 11, exp2 of an argument below 64 to 2^-21; sums and
                                # products in f32, 32 roundings at most; an fp16 output rounded once more
                                few = dtype == moert.F32 or 2 * n <= 16
                                rel = 2.0 ** -20 if few else 2.0 ** -11
                                if size * 1.4427 <= 2 ** 16:  # exponents of 2 round as the scores do, 4 times at most
                                    rel += 4 * 2.0 ** -24 * size
                                off = rel * np.abs(x[w]).mean(0) + 2.0 ** -24 * np.abs(x[w]).max()
                                if dtype == moert.F16:
                                    off = off + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
                                for a in (2 * h, 2 * h + 1):
                                    worst = np.abs(out[0, i, a].astype(np.float64) - want) / off
                                    assert (worst <= 1).all(), (kind, every, size, sign, i, a, float(worst.max()))
                        if decay is not None:
                            mass = np.stack([dev.mass(0, h, -(-rows // B)) for h in range(2)])
                            assert np.isfinite(mass).all() and (mass >= 0).all() and (mass <= 2 * n).all(), (kind, size)


def test_factors_of_a_score_that_leave_f32_together(hip):
    """Queries of 3e38 beside keys of 1e-6, scales from 1e-30 to 1e36: the scores are numbers, whatever two of their
    three factors make. All the weight is on the row of the largest one."""
    rng = np.random.default_rng(32)
    d, rows = 64, 300
    dev, ref = both(hip, 1, 1, d, 512)
    k, v = np.zeros((1, rows, 1, d), np.float32), normal(rng, 1, rows, 1, d)
    k[..., 0] = rng.integers(1, 100, (1, rows, 1)) * 2.0 ** -20
    k[0, 130, 0, 0] = 127 * 2.0 ** -20
    dev.append(k, v)
    ref.append(k, v)
    want = ref.rows(0, 0)[1][130]
    for n in (1, 20):
        for size, scale in ((3e38, 1e3), (3e38, 1.0), (3e38, 1e-30), (1e20, 1e15), (1e3, 1e36), (1e-3, 1e30)):
            q = np.zeros((1, n, 2, d), np.float32)
            q[..., 0] = size
            for out in (dev.attend(q, scale), dev.attend(q, scale, decay=0.5)):
                # two halves of a weight, scales and sums: 16 roundings at most
                assert (np.abs(out - want) <= 2.0 ** -20 * np.abs(want).max()).all(), (n, size, scale)


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("dtype", [moert.F32, moert.F16])
def test_subnormal_fp16_counts(hip, dtype, n):
    """Queries, rows of K and rows of V that fp16 holds as subnormals, coded and in the tail, with scales that make
    ordinary scores of them."""
    rng = np.random.default_rng(33)
    for rows in (20, 75):
        for size_q, size_k, size_v in ((2.0 ** -20, 1.0, 1.0), (1.0, 2.0 ** -20, 1.0), (1.0, 1.0, 2.0 ** -20),
                                       (2.0 ** -20, 2.0 ** -20, 2.0 ** -20)):
            dev, ref = both(hip, 1, 2, 64, 128)
            k, v = normal(rng, 1, rows, 2, 64, scale=size_k), normal(rng, 1, rows, 2, 64, scale=size_v)
            dev.append(k, v)
            ref.append(k, v)
            q = normal(rng, 1, n, 6, 64, scale=size_q).astype(np.float16)
            scale = float(np.float32(0.125 / (size_q * size_k)))
            want = ref.attend(q, scale)
            off = weights_bound(ref, q, scale, dtype == moert.F16)
            got = dev.attend(q, scale, dtype).astype(np.float64)
            assert (np.abs(got - want) <= off).all(), (rows, size_q, size_k, size_v, (np.abs(got - want) / off).max())
