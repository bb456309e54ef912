"""The paged K/V cache on the device against its definition in 64 bits (tests/pages_util.py): plans exactly, the pool bit
for bit, attention within bounds that follow from its roundings."""
import numpy as np
import pytest

import kv8_util as ku
import moert
import pages_util as pu
from pages_util import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip(gpu):
    h = ku.Hip()
    yield h
    h.close()


def both(hip, *shape, dtype=F16):
    return pu.Device(hip, *shape, dtype=dtype), pu.Cache(*shape, dtype=dtype)


def cache_type(dtype):
    return BF16 if dtype == BF16 else F16


def normal(rng, *shape, scale=1.0):
    return (scale * rng.standard_normal(shape)).astype(np.float32)


def step(dev, ref, rng, new, dtype, tokens=None, scale=1.0, k=None, v=None):
    """Plans and appends rows of every sequence, on both sides; the starts."""
    tokens = int(sum(max(n, 0) for n in new)) if tokens is None else tokens
    want = ref.plan(new, tokens)
    got, at = dev.plan(new, tokens)
    for a, b, name in zip(got, want, ("starts", "slots", "positions")):
        assert np.array_equal(a, b), name
    pu.assert_planned(dev, ref)
    if tokens:
        k = pu.to_bits(normal(rng, tokens, ref.H, ref.d, scale=scale) if k is None else k, dtype)
        v = pu.to_bits(normal(rng, tokens, ref.H, ref.d, scale=scale) if v is None else v, dtype)
        dev.append(k, v, at[1], dtype)
        ref.append(k, v, want[1], dtype)
    return want[0]


def queries(rng, dtype, *shape, scale=2.0):
    q = pu.to_bits(normal(rng, *shape, scale=scale), dtype)
    return q, pu.from_bits(q, dtype)


# ---- plans -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seqs,page,pages,max_pages,steps", [
    (1, 32, 1, 1, 6), (1, 256, 7, 5, 8), (5, 32, 16, 8, 12), (64, 64, 150, 16, 12), (1023, 32, 900, 9, 4),
    (1024, 128, 3000, 6, 4), (1025, 32, 2000, 40, 4), (3000, 64, 4000, 7, 4)])
def test_plans(hip, seqs, page, pages, max_pages, steps):
    """Step after step on the same cache: prompts and single rows, sequences that end, pages that run out, rows beyond
    max_pages and beyond the room for rows."""
    rng = np.random.default_rng(seqs + page)
    dev, ref = both(hip, seqs, 1, 64, page, pages, max_pages)
    pu.assert_planned(dev, ref)
    for i in range(steps):
        new = rng.choice([0, 1, 1, 1, -1, 3, page - 1, page, page + 1, 2 * page + 3], seqs)
        if i % 3 == 2:
            new[rng.integers(seqs)] = max_pages * page + 1  # never fits
        total = int(sum(max(n, 0) for n in new))
        tokens = [total, total + 37, max(0, total - 5), 0, total // 2][i % 5]
        want = ref.plan(new, tokens)
        got, _ = dev.plan(new, tokens, positions=i % 2 == 0)
        assert np.array_equal(got[0], want[0])
        assert np.array_equal(got[1], want[1])
        if i % 2 == 0:
            assert np.array_equal(got[2], want[2])
        pu.assert_planned(dev, ref)
    if any(ref.refused):
        with pytest.raises(moert.MoertError) as e:
            dev.c.lengths()
        assert e.value.code == moert.E_FULL and e.value.lengths.tolist() == ref.rows
    else:
        assert dev.c.lengths().tolist() == ref.rows
    assert dev.plan([-1] * seqs, 0) and dev.c.lengths().tolist() == [0] * seqs
    assert sorted(dev.array("free")[1:].tolist()) == list(range(pages)) and dev.array("free")[0] == pages


@pytest.mark.parametrize("tokens", [4095, 4096, 4097, 100001])
def test_plan_of_many_rows(hip, tokens):
    """One long prompt among short ones, on either side of where the rows' slots get a launch of their own."""
    dev, ref = both(hip, 9, 1, 64, 64, 1700, 1600)
    new = [1, 0, 2, tokens - 40, 0, 31, 1, 0, 0]
    for pad in (0, 5):
        want = ref.plan(new, tokens + pad)
        got, _ = dev.plan(new, tokens + pad)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        new = [1] * 9 if tokens > 4097 else [0, 1, 2, 3, 4, 5, 6, 7, 8]
    pu.assert_planned(dev, ref)


def test_plan_of_the_largest_requests(hip):
    """Requests of 2^31 - 1 rows are refused one by one, and their count stops at the type's largest number."""
    dev, ref = both(hip, 1030, 1, 64, 32, 8, 4)
    new = np.full(1030, 2 ** 31 - 1)
    new[[0, 700, 1029]] = 5, 6, 7
    for _ in range(2):
        want = ref.plan(new, 100)
        got, _ = dev.plan(new, 100)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        pu.assert_planned(dev, ref)


def test_plan_keeps_to_its_buffers_whatever_they_hold(hip):
    """Broken tables, states and free lists, with known bytes around every array."""
    rng = np.random.default_rng(3)
    seqs, page, pages, max_pages, tokens = 40, 32, 50, 6, 300
    shapes = moert.pages_shapes(seqs, 1, 64, page, pages, max_pages)
    sizes = {"table": seqs * max_pages, "state": seqs * 4, "free": pages + 1, "new": seqs, "starts": seqs + 1,
             "slots": tokens, "positions": tokens}
    assert int(np.prod(shapes["table"][0])) == sizes["table"]
    for i in range(12):
        whole, at, n = [], {}, 64
        for name, size in sizes.items():
            at[name] = n
            n += size + 64
        host = np.full(n, 0x5A5A5A5A, np.int32)
        for name in ("table", "state", "free"):
            host[at[name]:at[name] + sizes[name]] = rng.choice(
                [-2 ** 31, -1, 0, 1, 7, 49, 50, 191, 192, 193, 2 ** 20, 2 ** 31 - 1], sizes[name])
        host[at["new"]:at["new"] + seqs] = rng.choice([-5, -1, 0, 1, 33, 192, 193, 2 ** 31 - 1], seqs)
        if i % 2:
            host[at["free"]] = rng.integers(0, pages + 1)
        base = hip.upload(host)
        p = {name: base + 4 * a for name, a in at.items()}
        c = moert.Pages(seqs, 1, 64, page, pages, max_pages, {k: p[k] for k in ("table", "state", "free")})
        c.plan(p["new"], tokens, p["starts"], p["slots"], p["positions"])
        hip.sync()
        got = hip.get(base, (n,), np.int32)
        guard = np.ones(n, bool)
        for name, size in sizes.items():
            guard[at[name]:at[name] + size] = False
        assert (got[guard] == 0x5A5A5A5A).all()
        assert np.array_equal(got[at["new"]:at["new"] + seqs], host[at["new"]:at["new"] + seqs])
        starts = got[at["starts"]:at["starts"] + seqs + 1]
        assert (np.diff(starts) >= 0).all() and starts[0] == 0 and starts[-1] <= tokens
        slots = got[at["slots"]:at["slots"] + tokens]
        assert ((slots >= -1) & (slots < pages * page)).all()
        assert 0 <= got[at["free"]] <= pages
        whole.append(base)


# ---- rows ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_appends(hip, dtype, d, page):
    """Prompts and single rows of ragged sequences, blocks begun in one call and ended in others; rows behind the last
    are not written."""
    rng = np.random.default_rng(d + page)
    dev, ref = both(hip, 3, 2, d, page, 24, 8, dtype=cache_type(dtype))
    for new, pad in (([1, 37, 0], 3), ([31, 1, 5], 0), ([1, 1, 1], 1), ([70, 0, 131], 9), ([1, 0, 1], 0)):
        step(dev, ref, rng, new, dtype, tokens=sum(new) + pad)
        pu.assert_holds(dev, ref)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_slots_in_any_order_and_outside_the_pool(hip, dtype):
    rng = np.random.default_rng(1)
    dev, ref = both(hip, 1, 3, 64, 64, 9, 9, dtype=cache_type(dtype))
    slots = rng.permutation(9 * 64)[:301].astype(np.int64)
    slots[::7] = rng.choice([-1, -2 ** 31, 9 * 64, 9 * 64 + 1, 2 ** 31 - 1], slots[::7].size)
    k, v = (pu.to_bits(normal(rng, 301, 3, 64), dtype) for _ in range(2))
    dev.append(k, v, slots, dtype)
    ref.append(k, v, slots, dtype)
    pu.assert_holds(dev, ref)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shift,row,head", [(0, 3 * 64 + 8, 64), (1, 3 * 64 + 1, 64), (0, 64, 64 * 40), (0, 67, 67 * 40),
                                            (0, -200, 64), (4, 200, -64)])
def test_strides(hip, dtype, shift, row, head):
    """Rows with gaps, of odd strides, heads first, backwards, and from an odd element on."""
    rng = np.random.default_rng(2)
    n, H, d, item = 40, 3, 64, 4 if dtype == F32 else 2
    dev, ref = both(hip, 1, H, d, 32, 4, 4, dtype=cache_type(dtype))
    size = abs(row) * n + abs(head) * H + 500
    first = shift + (abs(row) * n if row < 0 else 0) + (abs(head) * H if head < 0 else 0)
    k, v = (pu.to_bits(normal(rng, size), dtype) for _ in range(2))
    at = first + np.arange(n)[:, None, None] * row + np.arange(H)[None, :, None] * head + np.arange(d)
    slots = rng.permutation(128)[:n]
    dev.c.append(hip.upload(k) + first * item, hip.upload(v) + first * item, hip.upload(slots.astype(np.int32)), n,
                 dtype=dtype, strides=(row, head))
    ref.append(k[at], v[at], slots, dtype)
    pu.assert_holds(dev, ref)
    # the same strides for queries and outputs
    heads = 3
    starts, ref.table[0], ref.rows[0] = [0, n], [0, 1, 2, 3], 128
    for s in range(128):
        if np.isnan(ref.k[s]).any():
            kk = pu.to_bits(normal(rng, 1, H, d), dtype)
            dev.append(kk, kk, [s], dtype)
            ref.append(kk, kk, [s], dtype)
    dev.set("table", [0, 1, 2, 3])
    dev.set("state", [128, 0, 128 - n, 0])
    out = np.full(size, 7.0, np.float32) if dtype == F32 else np.full(size, 0x4321, np.uint16)
    po = hip.upload(out)
    ws, ws_bytes = dev.workspace(heads, n)
    dev.c.prompt(hip.upload(k) + first * item, po + first * item, heads, 0.125, hip.upload(np.int32(starts)), n,
                 ws, ws_bytes, dtype=dtype, q_strides=(row, head), out_strides=(row, head)) if min(row, head) > 0 else None
    hip.sync()
    got = hip.get(po, out.shape, out.dtype)
    if min(row, head) > 0:
        pu.check(got[at], ref.attend(pu.from_bits(k[at], dtype), starts, 0.125, dtype), dtype)
        rest = np.ones(size, bool)
        rest[at.reshape(-1)] = False
        assert (got[rest] == pu.untouched(dtype)).all()


@pytest.mark.parametrize("dtype,big", [(F32, 65520.0), (F32, np.inf), (F32, np.nan), (F16, np.inf), (F16, np.nan),
                                       (BF16, -np.inf), (BF16, np.nan)])
def test_rows_that_are_not_finite(hip, dtype, big):
    """They make NaN of what sees them, in one KV head, and of nothing else."""
    rng = np.random.default_rng(4)
    dev, ref = both(hip, 2, 2, 64, 32, 12, 6, dtype=cache_type(dtype))
    k, v = normal(rng, 120, 2, 64), normal(rng, 120, 2, 64)
    k[50, 0, 3] = big
    v[70, 1, 60] = big
    starts = step(dev, ref, rng, [100, 20], dtype, k=k, v=v)
    pu.assert_holds(dev, ref)
    q, x = queries(rng, dtype, 120, 4, 64)
    want = ref.attend(x, starts, 0.125, dtype)
    assert np.isnan(want[0][50:100, :2]).all() and not np.isnan(want[0][:50]).any() and not np.isnan(want[0][100:]).any()
    pu.check(dev.prompt(q, 0.125, dtype, starts), want, dtype)
    q, x = queries(rng, dtype, 2, 4, 64)
    pu.check(dev.attend(q, 0.125, dtype), ref.attend(x, [0, 1, 2], 0.125, dtype), dtype)


# ---- attention of one position -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,g,d,page", [(1, 1, 64, 32), (2, 3, 64, 64), (1, 16, 128, 32), (2, 17, 64, 128),
                                        (1, 64, 128, 256), (8, 4, 128, 64)])
def test_attention_of_one_position(hip, dtype, H, g, d, page):
    """Lengths around blocks, pages and shares of waves, one without rows."""
    rng = np.random.default_rng(H + g + d)
    lens = [0, 1, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 300]
    dev, ref = both(hip, len(lens), H, d, page, 80, 300 // page + 2, dtype=cache_type(dtype))
    for part in (lens[:7] + [0] * 6, [0] * 7 + lens[7:]):  # pages of different sequences between each other
        step(dev, ref, rng, part, dtype)
    q, x = queries(rng, dtype, len(lens), H * g, d)
    starts = np.arange(len(lens) + 1)
    pu.check(dev.attend(q, d ** -0.5, dtype), ref.attend(x, starts, d ** -0.5, dtype), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("seqs,length,max_pages", [(1, 5000, 160), (1, 20011, 1024), (3, 2000, 64), (30, 700, 32),
                                                   (300, 90, 4)])
def test_long_and_many_sequences(hip, dtype, seqs, length, max_pages):
    """Few long sequences, whose cache is split over workgroups, and many short ones."""
    rng = np.random.default_rng(seqs)
    lens = [max(1, length - 7 * s) for s in range(seqs)]
    page = 32
    dev, ref = both(hip, seqs, 2, 64, page, sum(-(-n // page) for n in lens) + 1, max_pages, dtype=cache_type(dtype))
    step(dev, ref, rng, lens, dtype)
    q, x = queries(rng, dtype, seqs, 6, 64)
    pu.check(dev.attend(q, 0.125, dtype), ref.attend(x, np.arange(seqs + 1), 0.125, dtype), dtype)


def test_only_sequences_of_one_row_are_attended(hip):
    """Idle sequences, prompts and rows behind the last stay as they were; the prompt with least = 2 takes the others."""
    rng = np.random.default_rng(7)
    dev, ref = both(hip, 6, 2, 64, 32, 60, 10)
    step(dev, ref, rng, [40, 1, 33, 0, 5, 100], F32)
    starts = step(dev, ref, rng, [1, 0, 7, 0, 1, 1], F32, tokens=14)
    q, x = queries(rng, F32, 14, 6, 64)
    want = ref.attend(x, starts, 0.125, F32, which=lambda n: n == 1)
    assert want[2].sum() == 3
    pu.check(dev.attend(q, 0.125, F32, starts=starts), want, F32)
    for least in (1, 2, 7, 8):
        pu.check(dev.prompt(q, 0.125, F32, starts, least=least),
                 ref.attend(x, starts, 0.125, F32, which=lambda n: n >= least), F32)


# ---- prompts -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,g,d,page", [(1, 1, 64, 32), (2, 3, 64, 64), (1, 5, 128, 32), (2, 8, 128, 256),
                                        (1, 64, 64, 32), (1, 33, 128, 64)])
def test_prompts(hip, dtype, H, g, d, page):
    """Ragged prompts in one batch, after nothing and after rows of other lengths; then a second part of each."""
    rng = np.random.default_rng(H + g + d)
    new = [1, 2, 0, 31, 32, 33, 65, 100]
    dev, ref = both(hip, len(new), H, d, page, 60, 400 // page + 2, dtype=cache_type(dtype))
    for part, pad in ((new, 3), ([64, 1, 17, 0, 1, 32, 31, 40], 0)):
        starts = step(dev, ref, rng, part, dtype, tokens=sum(part) + pad)
        q, x = queries(rng, dtype, sum(part) + pad, H * g, d)
        pu.check(dev.prompt(q, d ** -0.5, dtype, starts), ref.attend(x, starts, d ** -0.5, dtype), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_long_prompts(hip, dtype, d):
    rng = np.random.default_rng(d)
    dev, ref = both(hip, 3, 1, d, 64, 60, 30, dtype=cache_type(dtype))
    step(dev, ref, rng, [0, 611, 30], dtype)
    starts = step(dev, ref, rng, [700, 129, 301], dtype)
    q, x = queries(rng, dtype, 1130, 2, d)
    pu.check(dev.prompt(q, d ** -0.5, dtype, starts), ref.attend(x, starts, d ** -0.5, dtype), dtype)


def test_positions_that_see_nothing(hip):
    """Fewer rows than queries: the first queries see nothing and get 0, as do all of a refused sequence."""
    rng = np.random.default_rng(9)
    dev, ref = both(hip, 3, 2, 64, 32, 5, 5)
    step(dev, ref, rng, [60, 40, 3], F32)
    starts = step(dev, ref, rng, [30, 0, 200], F32)  # the first and the last are refused: no page is left
    assert ref.first == [-1, 40, -1]
    q, x = queries(rng, F32, 230, 4, 64)
    got = dev.prompt(q, 0.125, F32, starts)
    assert not got.any()
    ref.first = [0, 0, 0]
    dev.set("state", [[60, 0, 0, 0], [40, 0, 0, 0], [3, 0, 0, 0]])
    want = ref.attend(x, [0, 100, 223, 230], 0.125, F32)
    assert not want[0][:40].any() and want[0][40:100].any()
    pu.check(dev.prompt(q, 0.125, F32, [0, 100, 223, 230]), want, F32)


# ---- numbers -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30, 3.0])
def test_scales(hip, dtype, scale):
    rng = np.random.default_rng(11)
    dev, ref = both(hip, 2, 1, 64, 32, 20, 10, dtype=cache_type(dtype))
    starts = step(dev, ref, rng, [75, 200], dtype)
    q, x = queries(rng, dtype, 275, 2, 64, scale=1.0)
    pu.check(dev.prompt(q, scale, dtype, starts), ref.attend(x, starts, scale, dtype), dtype)
    q, x = queries(rng, dtype, 2, 2, 64, scale=1.0)
    pu.check(dev.attend(q, scale, dtype), ref.attend(x, [0, 1, 2], scale, dtype), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["subnormal", "large", "far", "falling", "rising", "equal", "tiny_q", "huge_q"])
def test_extremes(hip, dtype, kind):
    """Values at the ends of their types; scores that fall or rise all along; equal ones beyond what f32 tells apart."""
    if dtype != F32 and kind in ("tiny_q", "huge_q"):
        return
    rng = np.random.default_rng(13)
    n = 150
    dev, ref = both(hip, 1, 1, 64, 32, 6, 6, dtype=cache_type(dtype))
    k, v, q, scale = normal(rng, n, 1, 64), normal(rng, n, 1, 64), normal(rng, n, 2, 64), 0.125
    if kind == "subnormal":
        k, v, q, scale = k * 3e-6, v * 3e-6, q * 3e-6, 1e10
    elif kind == "large":
        k, v = np.clip(k, -1, 1) * 60000, np.clip(v * 4, -1, 1) * 65504
        q, scale = q * 1e3, 1e-8
    elif kind == "far":
        k, q, scale = k * 200, q * 200, 1.0
    elif kind in ("falling", "rising"):
        k = np.broadcast_to(np.linspace(0, 30, n, dtype=np.float32)[:, None, None], k.shape).copy()
        k = k[::-1] if kind == "falling" else k
        q, scale = np.full_like(q, 1.0), 1.0
    elif kind == "equal":
        k, q, scale = np.full_like(k, 300.0), np.full_like(q, 500.0), 1000.0
    elif kind == "tiny_q":
        q, scale = q * 1e-35, 1e34
    elif kind == "huge_q":
        q, scale = q * 1e30, 1e-31
    starts = step(dev, ref, rng, [n], dtype, k=k, v=v)
    b = pu.to_bits(q, dtype)
    x = pu.from_bits(b, dtype)
    if kind == "equal":
        out, off, wrote = ref.attend(x, starts, 0.0, dtype)  # equal scores of any size weigh the same
    else:
        out, off, wrote = ref.attend(x, starts, scale, dtype)
    pu.check(dev.prompt(b, scale, dtype, starts), (out, off, wrote), dtype)
    last = (out[-1:], off[-1:], wrote[-1:])
    pu.check(dev.attend(b[-1:], scale, dtype), last, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_queries_that_are_not_finite(hip, dtype):
    rng = np.random.default_rng(15)
    dev, ref = both(hip, 3, 1, 64, 32, 20, 10, dtype=cache_type(dtype))
    starts = step(dev, ref, rng, [40, 9, 0], dtype)
    for big in (np.inf, -np.inf, np.nan):
        q = normal(rng, 49, 2, 64)
        q[7, 1, 5] = q[45, 0, 63] = big
        b = pu.to_bits(q, dtype)
        pu.check(dev.prompt(b, 0.125, dtype, starts), ref.attend(pu.from_bits(b, dtype), starts, 0.125, dtype), dtype)
        b = b[[7, 45, 7]]  # the last sees nothing
        pu.check(dev.attend(b, 0.125, dtype), ref.attend(pu.from_bits(b, dtype), range(4), 0.125, dtype), dtype)


# ---- calls ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_server(hip, dtype):
    """Plans, rows, prompts and decoding steps as they would be used, in a captured graph of a step, replayed with eager
    work in between; sequences end and others take their pages. Outputs may lie over the queries."""
    rng = np.random.default_rng(17)
    S, H, heads, d, T = 4, 2, 6, 64, 80
    t = np.float32 if dtype == F32 else np.uint16
    dev, ref = both(hip, S, H, d, 32, 14, 8, dtype=cache_type(dtype))
    new, starts, slots, pos = (hip.upload(np.zeros(n, np.int32)) for n in (S, S + 1, T, T))
    k, v, q = (hip.upload(np.zeros((T, n, d), t)) for n in (H, H, heads))
    ws, size = dev.workspace(heads, T)
    stream = hip.stream()

    def calls():
        dev.c.plan(new, T, starts, slots, pos, stream=stream)
        dev.c.append(k, v, slots, T, dtype=dtype, stream=stream)
        dev.c.prompt(q, q, heads, 0.125, starts, T, ws, size, least=2, dtype=dtype, stream=stream)
        dev.c.attend(q, q, heads, 0.125, ws, size, starts=starts, tokens=T, dtype=dtype, stream=stream)

    graph = hip.capture(stream, calls)
    for n, want in enumerate([[70, 5, 0, 1], [1, 1, 1, 1], [1, -1, 33, 0], [0, 64, 1, 1], [1, 1, -1, -1], [60, 1, 0, 9]]):
        hip.put(new, np.array(want, np.int32))
        kk, vv = (pu.to_bits(normal(rng, T, H, d), dtype) for _ in range(2))
        qq, x = queries(rng, dtype, T, heads, d)
        for at, a in ((k, kk), (v, vv), (q, qq)):
            hip.put(at, a)
        hip.sync()
        if n % 3 == 1:
            calls()
        else:
            hip.launch(graph, stream)
        hip.sync()
        at, sl, po = ref.plan(want, T)
        ref.append(kk, vv, sl, dtype)
        pu.assert_planned(dev, ref)
        assert np.array_equal(hip.get(starts, (S + 1,), np.int32), at)
        assert np.array_equal(hip.get(slots, (T,), np.int32), sl)
        assert np.array_equal(hip.get(pos, (T,), np.int32), po)
        pu.assert_holds(dev, ref)
        out, off, wrote = ref.attend(x, at, 0.125, dtype)
        got = hip.get(q, (T, heads, d), t)
        assert np.array_equal(got[~wrote], qq[~wrote])
        got[~wrote] = pu.untouched(dtype)
        pu.check(got, (out, off, wrote), dtype)


def test_calls_give_the_same_bits_again(hip):
    """Twice on one stream, and at once on two with a workspace each."""
    rng = np.random.default_rng(19)
    for dtype in (F32, F16, BF16):
        dev, ref = both(hip, 3, 2, 64, 32, 120, 64, dtype=cache_type(dtype))
        starts = step(dev, ref, rng, [900, 333, 1500], dtype)
        q, _ = queries(rng, dtype, 2733, 6, 64)
        assert np.array_equal(dev.prompt(q, 0.125, dtype, starts), dev.prompt(q, 0.125, dtype, starts))
        first = dev.attend(q[:3], 0.125, dtype)
        assert np.array_equal(first, dev.attend(q[:3], 0.125, dtype))
        outs = []
        at = hip.upload(q[:3])
        for _ in range(2):
            s, (ws, size), out = hip.stream(), dev.workspace(6), dev._out(q[:3], dtype)
            hip.sync()
            for _ in range(5):
                dev.c.attend(at, out, 6, 0.125, ws, size, dtype=dtype, stream=s)
            outs.append(out)
        hip.sync()
        for out in outs:
            assert np.array_equal(first, hip.get(out, (3, 6, 64), q.dtype))


def test_broken_tables_stay_inside_the_buffers(hip):
    """Tables, states, starts and slots of any value: no output outside its rows, no fault."""
    rng = np.random.default_rng(21)
    wild = [-2 ** 31, -1, 0, 1, 5, 6, 31, 32, 200, 2 ** 20, 2 ** 31 - 1]
    for dtype in (F32, BF16):
        dev, ref = both(hip, 5, 2, 64, 32, 6, 6, dtype=cache_type(dtype))
        k = pu.to_bits(normal(rng, 192, 2, 64), dtype)
        dev.append(k, k, np.arange(192), dtype)
        for i in range(10):
            dev.set("table", rng.choice(wild, 30))
            dev.set("state", rng.choice(wild, 20))
            starts = np.sort(rng.choice(wild, 6)) if i % 2 else rng.choice(wild, 6)
            q, _ = queries(rng, dtype, 40, 4, 64)
            for call in (dev.prompt, dev.attend):
                got = call(q, 0.125, dtype, starts=starts)
                assert not np.isnan(pu.from_bits(got, dtype)).any()
            dev.append(k, k, rng.choice(wild, 192), dtype)
            dev.append(k, k, np.arange(192), dtype)


def test_far_offsets(hip):
    """A pool of 5 GB: rows at its end, beyond 2^32 bytes and 2^31 elements."""
    rng = np.random.default_rng(23)
    H, d, page = 8, 128, 256
    pages = 5 * 2 ** 30 // (H * page * d * 2)
    dev = pu.Device(hip, 1, H, d, page, pages, 3, fill=False)
    ref = pu.Cache(1, H, d, page, 3, 3)
    high = np.array([pages - 1, 0, pages - 2])
    n = 600
    k, v = (pu.to_bits(normal(rng, n, H, d), F16) for _ in range(2))
    at = np.arange(n)
    dev.append(k, v, high[at // page] * page + at % page, F16)
    ref.append(k, v, at, F16)
    ref.table[0], ref.rows[0] = [0, 1, 2], n
    dev.set("table", high)
    dev.set("state", [n, 0, 0, 0])
    q, x = queries(rng, F16, 5, 8, d)
    pu.check(dev.prompt(q, 0.09, F16, [0, 5]), ref.attend(x, [0, 5], 0.09, F16), F16)
    pu.check(dev.attend(q[:1], 0.09, F16), ref.attend(x[:1], [0, 1], 0.09, F16), F16)


def test_calls_of_no_rows(hip):
    dev, ref = both(hip, 2, 1, 64, 32, 4, 2)
    step(dev, ref, np.random.default_rng(1), [0, 0], F32)
    z = np.zeros((0, 1, 64), np.float32)
    dev.append(z, z, [0], F32)
    dev.prompt(z, 0.125, F32, [0, 0, 0])
    assert dev.attend(z, 0.125, F32, starts=[0, 0, 0]).size == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_before_the_first_sequence(hip, dtype):
    """Starts that begin behind rows of no sequence: those stay as they were."""
    rng = np.random.default_rng(25)
    for n, before in ((200, 100), (9, 40), (1, 7)):
        dev, ref = both(hip, 3, 2, 64, 32, 40, 12, dtype=cache_type(dtype))
        step(dev, ref, rng, [n, 0, n + 3], dtype)
        starts = before + np.array([0, n, n, 2 * n + 3])
        q, x = queries(rng, dtype, starts[-1] + 5, 6, 64)
        pu.check(dev.prompt(q, 0.125, dtype, starts), ref.attend(x, starts, 0.125, dtype), dtype)
        starts = before + np.array([0, 1, 1, 2])
        pu.check(dev.attend(q, 0.125, dtype, starts=starts), ref.attend(x, starts, 0.125, dtype), dtype)


@pytest.mark.parametrize("tokens", [3, 40, 700])
def test_broken_starts_write_nothing_outside_the_rows(hip, tokens):
    """Known bytes before and behind the outputs of a batch, in whose starts is anything."""
    rng = np.random.default_rng(tokens)
    dev, ref = both(hip, 9, 2, 64, 32, 40, 30)
    k = pu.to_bits(normal(rng, 40 * 32, 2, 64), F16)
    dev.append(k, k, np.arange(40 * 32), F16)
    dev.set("table", rng.integers(0, 40, 9 * 30))
    dev.set("state", np.stack([rng.integers(0, 960, 9), np.zeros(9), np.zeros(9), np.zeros(9)], 1))
    pad, row = 5000 * 4 * 64, 4 * 64
    ws, size = dev.workspace(4, tokens)
    q = hip.upload(pu.to_bits(normal(rng, tokens * row + 2 * pad), F16)) + 2 * pad
    for i in range(12):
        starts = rng.choice([-2 ** 31, -1, 0, 1, 2, tokens // 2, tokens - 1, tokens, tokens + 1, 2 ** 31 - 1], 10)
        out = hip.upload(np.full(tokens * row + 2 * pad, 0x4321, np.uint16))
        at = hip.upload(starts.astype(np.int32))
        dev.c.prompt(q, out + 2 * pad, 4, 0.125, at, tokens, ws, size)
        dev.c.attend(q, out + 2 * pad, 4, 0.125, ws, size, starts=at, tokens=tokens)
        hip.sync()
        got = hip.get(out, (tokens * row + 2 * pad,), np.uint16)
        assert (got[:pad] == 0x4321).all() and (got[-pad:] == 0x4321).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q_strides,out_strides", [((4 * 64 + 1, 64), (4 * 64, 64)), ((4 * 64, 64), (300, 67)),
                                                   ((-4 * 64, 64), (64, 64 * 50))])
def test_strides_of_queries_and_outputs(hip, dtype, q_strides, out_strides):
    """Each with its own, of one position and of prompts."""
    rng = np.random.default_rng(27)
    n, heads, d, item = 46, 4, 64, 4 if dtype == F32 else 2
    dev, ref = both(hip, 3, 2, d, 32, 12, 8, dtype=cache_type(dtype))
    starts = step(dev, ref, rng, [40, 5, 1], dtype)

    def places(strides):
        first = max(0, -strides[0]) * n
        return first, first + np.arange(n)[:, None, None] * strides[0] + np.arange(heads)[None, :, None] * strides[1] + np.arange(d)

    (q0, q_at), (o0, o_at) = places(q_strides), places(out_strides)
    q = pu.to_bits(normal(rng, q_at.max() + 9, scale=2.0), dtype)
    ws, size = dev.workspace(heads, n)
    for call, which in (("prompt", lambda m: m >= 1), ("attend", lambda m: m == 1)):
        out = np.full(o_at.max() + 9, pu.untouched(dtype))
        at = hip.upload(out)
        kw = dict(starts=hip.upload(starts.astype(np.int32)), tokens=n, ws=ws, ws_bytes=size, dtype=dtype,
                  q_strides=q_strides, out_strides=out_strides)
        getattr(dev.c, call)(hip.upload(q) + q0 * item, at + o0 * item, heads, 0.125, **kw)
        hip.sync()
        got = hip.get(at, out.shape, out.dtype)
        pu.check(got[o_at], ref.attend(pu.from_bits(q[q_at], dtype), starts, 0.125, dtype, which), dtype)
        rest = np.ones(out.size, bool)
        rest[o_at.reshape(-1)] = False
        assert (got[rest] == pu.untouched(dtype)).all()


@pytest.mark.parametrize("new", [3, 40])
def test_prompts_of_many_sequences(hip, new):
    """More sequences than a wave looks at together, many of them without rows: few rows each, and more."""
    rng = np.random.default_rng(new)
    S = 150
    dev, ref = both(hip, S, 1, 64, 32, 400, 5)
    step(dev, ref, rng, rng.integers(0, 40, S), F16)
    counts = np.where(rng.random(S) < 0.5, 0, rng.integers(1, new + 1, S))
    starts = step(dev, ref, rng, counts, F16, tokens=int(counts.sum()) + 9)
    q, x = queries(rng, F16, int(counts.sum()) + 9, 3, 64)
    pu.check(dev.prompt(q, 0.125, F16, starts), ref.attend(x, starts, 0.125, F16), F16)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_batch_in_which_one_sequence_is_long(hip, dtype):
    """Few rows on average, but one prompt among single rows, and the other way round: whatever the choice, the same."""
    rng = np.random.default_rng(29)
    dev, ref = both(hip, 20, 1, 64, 32, 60, 20, dtype=cache_type(dtype))
    step(dev, ref, rng, [20] * 20, dtype)
    for new in ([300] + [1] * 19, [1] * 19 + [100]):
        starts = step(dev, ref, rng, new, dtype)
        q, x = queries(rng, dtype, sum(new), 2, 64)
        pu.check(dev.prompt(q, 0.125, dtype, starts), ref.attend(x, starts, 0.125, dtype), dtype)


# ---- scores of any size ----------------------------------------------------------------------------------------------
def one_sequence(hip, dtype, k, v, max_pages=None):
    """A cache of one sequence with the given rows (f32 values)."""
    rows, H, d = k.shape
    pages = -(-rows // 64)
    dev, ref = both(hip, 1, H, d, 64, pages, max_pages or pages, dtype=cache_type(dtype))
    step(dev, ref, np.random.default_rng(0), [rows], dtype, k=k.astype(np.float32), v=v.astype(np.float32))
    return dev, ref


def both_ways(dev, q, scale, dtype):
    """The last positions' outputs, of prompts of few rows and of many (with the queries behind others), and of the last
    position alone."""
    n = q.shape[0]
    yield n, dev.prompt(q, scale, dtype, [0, n])
    more = np.concatenate([np.repeat(q[:1], 60, 0), q])
    yield n, dev.prompt(more, scale, dtype, [0, 60 + n])[60:]
    yield 1, dev.attend(q[-1:], scale, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("max_pages", [11, 256])
def test_scores_of_any_size(hip, dtype, max_pages):
    """Scores of 10^4 to 10^30, far beyond the steps of exponents: all the weight on one row, or shared by every 37th in
    equal parts."""
    rng = np.random.default_rng(31)
    d, rows, n = 64, 700, 12
    v = normal(rng, rows, 2, d)
    for every in (rows, 37):
        k = np.zeros((rows, 2, d), np.float32)
        k[..., 0], k[..., 1] = rng.integers(20, 100, (rows, 2)), 127.0
        k[20::every, :, 0] = 127.0
        dev, ref = one_sequence(hip, dtype, k, v, max_pages)
        at = np.arange(20, rows, every)
        for size in (1e4, 1e5, 1e6, 1e7, 1e9, 1e12, 1e30):
            for sign in (1.0, -1.0):
                q = np.zeros((n, 4, d), np.float32)
                q[..., 0] = 16.0
                if sign < 0:  # every score below 0, the same ones apart
                    q[..., 1] = -32.0
                for m, out in both_ways(dev, pu.to_bits(q, dtype), size / (16.0 * 127.0), dtype):
                    for i in range(m):
                        for a in range(4):
                            x = ref.kv(0, a // 2, rows)[1][at[at < rows - m + 1 + i]]
                            want = x.mean(0)
                            # weights of one size, rounded alike; sums and products in f32, the output
                            off = 2.0 ** -19 * np.abs(x).mean(0) + pu.HALF[dtype] * (np.abs(want) + 2.0 ** -13)
                            if dtype == BF16:  # two numbers of 8 bits
                                off = off + 2.0 ** -15 * np.abs(x).mean(0)
                            err = np.abs(pu.from_bits(out, dtype)[i, a] - want)
                            assert (err <= off).all(), (every, size, sign, m, i, a, (err / off).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_near_f32s_lowest(hip, dtype):
    """Scores of about -1e36, apart by 1e34 and more: all the weight is on the least negative one that is seen."""
    rng = np.random.default_rng(33)
    d, rows = 64, 500
    k, v = np.zeros((rows, 1, d)), normal(rng, rows, 1, d)
    k[..., 0] = 127.0
    k[340, 0, 0] = 100.0
    dev, ref = one_sequence(hip, dtype, k, v)
    q = np.zeros((9, 2, d), np.float32)
    q[..., 0] = -1e34
    want = ref.kv(0, 0, rows)[1][340]
    for _, out in both_ways(dev, pu.to_bits(q, dtype), 1.0, dtype):
        assert (np.abs(pu.from_bits(out, dtype) - want) <= (pu.HALF[dtype] + 2.0 ** -22) * np.abs(want)).all()


def test_factors_of_a_score_that_leave_f32_together(hip):
    """Queries of 3e38 beside keys of 1e-6, scales from 1e-30 to 1e36: the scores are numbers, whatever two of their
    three factors make. All the weight is on the row of the largest one."""
    rng = np.random.default_rng(35)
    d, rows = 64, 300
    k, v = np.zeros((rows, 1, d)), normal(rng, rows, 1, d)
    k[..., 0] = rng.integers(1, 100, (rows, 1)) * 2.0 ** -20
    k[130, 0, 0] = 127 * 2.0 ** -20
    dev, ref = one_sequence(hip, F32, k, v)
    want = ref.kv(0, 0, rows)[1][130]
    for size, scale in ((3e38, 1e3), (3e38, 1.0), (3e38, 1e-30), (1e20, 1e15), (1e3, 1e36), (1e-3, 1e30)):
        q = np.zeros((9, 2, d), np.float32)
        q[..., 0] = size
        for _, out in both_ways(dev, q, scale, F32):
            assert (np.abs(out - want) <= 2.0 ** -20 * np.abs(want)).all(), (size, scale)


@pytest.mark.parametrize("max_pages", [6, 200])
def test_the_largest_values_stay_finite(hip, max_pages):
    """V of fp16's largest magnitude, weights whose rounding to fp16 has one sign in all rows that count."""
    d, rows = 64, 384
    k, v = np.zeros((rows, 1, d)), np.full((rows, 1, d), 65504.0)
    k[rows // 2:, :, 0] = 1.0
    v[..., 1::2] = -65504.0
    dev, ref = one_sequence(hip, F16, k, v, max_pages)
    q = np.zeros((3, 64, d), np.float32)
    q[..., 0] = 0.7 + np.arange(64) / 14.5
    for m, out in both_ways(dev, pu.to_bits(q, F16), 1.0, F16):
        got = pu.from_bits(out, F16)
        assert np.isfinite(got).all() and (np.abs(got - v[0, 0]) <= 65504.0 * 2.0 ** -11).all()


@pytest.mark.parametrize("size_q,size_k,size_v", [(2.0 ** -20, 1.0, 1.0), (1.0, 2.0 ** -20, 1.0), (1.0, 1.0, 2.0 ** -20),
                                                  (2.0 ** -20,) * 3])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_subnormal_fp16_counts(hip, dtype, size_q, size_k, size_v):
    rng = np.random.default_rng(37)
    rows, n = 200, 9
    dev, ref = one_sequence(hip, dtype, normal(rng, rows, 2, 64, scale=size_k), normal(rng, rows, 2, 64, scale=size_v))
    q = pu.to_bits(normal(rng, n, 6, 64, scale=size_q), dtype)
    scale = float(np.float32(0.125 / (size_q * size_k)))
    for m, out in both_ways(dev, q, scale, dtype):
        want = ref.attend(pu.from_bits(q[-m:], dtype), [0, m], scale, dtype)
        pu.check(out, want, dtype)


# ---- more calls ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_outputs_in_place_of_the_queries(hip, dtype):
    """out = q, of the same strides: every row of q is read before its output is written, with and without splits."""
    rng = np.random.default_rng(39)
    for max_pages in (20, 300):
        dev, ref = both(hip, 2, 2, 64, 32, 60, max_pages, dtype=cache_type(dtype))
        step(dev, ref, rng, [500, 333], dtype)
        ws, size = dev.workspace(6, 400)
        for starts in ([0, 5, 9], [0, 150, 300]):
            q, _ = queries(rng, dtype, starts[-1], 6, 64)
            want, at = dev.prompt(q, 0.125, dtype, starts), hip.upload(q)
            dev.c.prompt(at, at, 6, 0.125, hip.upload(np.int32(starts)), len(q), ws, size, dtype=dtype)
            hip.sync()
            assert np.array_equal(hip.get(at, q.shape, q.dtype), want)
        q, _ = queries(rng, dtype, 2, 6, 64)
        want, at = dev.attend(q, 0.125, dtype), hip.upload(q)
        dev.c.attend(at, at, 6, 0.125, ws, size, dtype=dtype)
        hip.sync()
        assert np.array_equal(hip.get(at, q.shape, q.dtype), want)


def test_two_graphs_of_one_cache_and_workspace(hip):
    """A step of single rows and one of prompts, captured apart, replayed in turn with eager work in between."""
    rng = np.random.default_rng(41)
    S, H, heads, d, T = 3, 1, 4, 64, 150
    dev, ref = both(hip, S, H, d, 32, 64, 128, dtype=F16)
    new, starts, slots = (hip.upload(np.zeros(n, np.int32)) for n in (S, S + 1, T))
    rows, q, out = (hip.upload(np.zeros((T, n, d), np.uint16)) for n in (H, heads, heads))
    ws, size = dev.workspace(heads, T)
    stream = hip.stream()

    def calls(single):
        dev.c.plan(new, T, starts, slots, stream=stream)
        dev.c.append(rows, rows, slots, T, stream=stream)
        if single:
            dev.c.attend(q, out, heads, 0.125, ws, size, starts=starts, tokens=T, stream=stream)
        else:
            dev.c.prompt(q, out, heads, 0.125, starts, T, ws, size, stream=stream)

    graphs = [hip.capture(stream, lambda: calls(single)) for single in (False, True)]
    for want in ([100, 1, 40], [1, 1, 1], [1, 0, 1], [20, 60, 0], [1, 1, 1], [0, 1, 1], [50, 50, 50]):
        single = max(want) == 1
        kk = pu.to_bits(normal(rng, T, H, d), F16)
        qq, x = queries(rng, F16, T, heads, d)
        hip.put(new, np.array(want, np.int32)), hip.put(rows, kk), hip.put(q, qq)
        hip.put(out, np.full((T, heads, d), 0x4321, np.uint16))
        hip.sync()
        hip.launch(graphs[single], stream)
        hip.sync()
        at, sl, _ = ref.plan(want, T)
        ref.append(kk, kk, sl, F16)
        pu.assert_planned(dev, ref)
        pu.check(hip.get(out, (T, heads, d), np.uint16), ref.attend(x, at, 0.125, F16), F16)
        assert dev.attend(qq[:3], 0.125, F16).size  # eager work on the default stream in between


def test_lengths_are_not_read_under_capture(hip):
    dev, _ = both(hip, 1, 1, 64, 32, 2, 2)
    stream = hip.stream()
    with pytest.raises(moert.MoertError) as e:
        hip.capture(stream, lambda: dev.c.lengths(stream=stream))
    assert "captured" in str(e.value)


def test_the_most_sequences_and_the_longest(hip):
    """65535 sequences in one plan; one sequence of 2^20 rows."""
    rng = np.random.default_rng(43)
    dev, ref = both(hip, 65535, 1, 64, 32, 50000, 3)
    few = np.where(np.arange(65535) % 200 == 7, 1, 0)  # 256 rows of thousands of sequences
    for new in (few, rng.choice([0, 0, 1, 33], 65535), few, rng.choice([-1, 0, 1, 40], 65535)):
        tokens = int(np.maximum(new, 0).sum()) + 5
        want = ref.plan(new, tokens)
        got, _ = dev.plan(new, tokens)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        pu.assert_planned(dev, ref)
    dev, ref = both(hip, 2, 1, 64, 256, 5000, 4096)
    for new in ([2 ** 20, 5], [1, 1], [-1, 0]):
        tokens = max(0, new[0]) + max(0, new[1])
        want = ref.plan(new, tokens)
        got, _ = dev.plan(new, tokens)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
        pu.assert_planned(dev, ref)
