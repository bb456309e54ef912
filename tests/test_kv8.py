"""The 8-bit K/V cache without a device: every refusal comes before anything is launched, the buffers' shapes, the
layout of a block of V, and the definition that the GPU tests compare with (tests/kv8_util.py) against plain facts."""
import math

import numpy as np
import pytest

import kv8_util as ku
import moert

GOOD = dict(seqs=2, kv_heads=2, head_dim=64, max_len=96)


def cache(buffers=None, **kw):
    c = {**GOOD, **kw}
    names = [n[:-4] for n, _ in moert.moert_kv8._fields_[4:]]
    at = {n: 0x10000 for n in names}  # never reached
    at.update(buffers or {})
    return moert.Kv8(c["seqs"], c["kv_heads"], c["head_dim"], c["max_len"], at)


CALLS = {
    "clear": lambda c, **kw: c.clear(**kw),
    "append": lambda c, **kw: c.append(**{**dict(k=0x20000, v=0x20000, n=1), **kw}),
    "attend": lambda c, **kw: c.attend(**{**dict(q=0x20000, out=0x20000, heads=4, n=1, scale=0.125, ws=0x30000,
                                                 ws_bytes=1 << 30), **kw}),
    "evict": lambda c, **kw: c.evict(**{**dict(keep=2), **kw}),
    "read": lambda c, **kw: c.read(**{**dict(k=0x20000, v=0x28000, pos=0, n=1), **kw}),
    "lengths": lambda c, **kw: c.lengths(**kw),
}


def refused(call, what):
    with pytest.raises(moert.MoertError) as e:
        call()
    assert e.value.code == moert.E_CONFIG, e.value
    assert what in str(e.value), e.value


@pytest.mark.parametrize("name", sorted(CALLS))
def test_bad_caches_are_refused(name):
    call = CALLS[name]
    for bad in (dict(seqs=0), dict(seqs=65536), dict(kv_heads=0), dict(kv_heads=257), dict(seqs=8192, kv_heads=129), dict(head_dim=32),
                dict(head_dim=96), dict(max_len=0), dict(max_len=95), dict(max_len=(1 << 20) + 32)):
        refused(lambda: call(cache(**bad), seq0=0, n_seqs=1), "kv8_" + name)
    for buf in ("k_codes", "v_codes", "k_scale", "v_scale", "k_tail", "v_tail", "tail_bad", "table", "state"):
        refused(lambda: call(cache({buf: None})), "null buffer")
        refused(lambda: call(cache({buf: 0x10002})), "aligned")
    for seqs in (dict(seq0=-1, n_seqs=1), dict(seq0=2, n_seqs=1), dict(seq0=0, n_seqs=3), dict(seq0=1, n_seqs=2),
                 dict(seq0=0, n_seqs=0), dict(seq0=0, n_seqs=-1), dict(seq0=2 ** 31 - 1, n_seqs=2 ** 31 - 1)):
        refused(lambda: call(cache(), **seqs), "sequences")


def test_a_cache_that_is_not_device_memory_is_refused():
    host = np.zeros(1 << 16, np.uint8)
    at = host.ctypes.data + -host.ctypes.data % 16
    bufs = {n[:-4]: at for n, _ in moert.moert_kv8._fields_[4:]}
    for call in CALLS.values():
        refused(lambda: call(cache(bufs)), "not in device memory")


def test_a_null_cache_and_unknown_buffers_are_refused():
    assert moert.lib().moert_kv8_clear(None, 0, 1, None) == moert.E_CONFIG
    with pytest.raises(ValueError):
        cache({"keys": 1})


def test_bad_rows_are_refused():
    c = cache()
    for n in (0, -1, 97):
        refused(lambda: CALLS["append"](c, n=n), "rows")
    for name in ("append", "read"):
        for kv in ("k", "v"):
            refused(lambda: CALLS[name](c, **{kv: None}), "null rows")
            refused(lambda: CALLS[name](c, **{kv: 0x20002}), "not aligned")
            refused(lambda: CALLS[name](c, dtype=moert.F16, **{kv: 0x20001}), "not aligned")
        for dtype in (moert.Q8_0, moert.Q4_0, 4, -1):
            refused(lambda: CALLS[name](c, dtype=dtype), "dtype")
    for pos, n in ((0, 0), (0, -3), (0, 97), (96, 1), (-97, 1)):
        refused(lambda: CALLS["read"](c, pos=pos, n=n), "positions")
    refused(lambda: CALLS["read"](c, v=0x20000), "one address")
    # rows to be written must not overlap, in whatever order the axes lie
    for strides in ((0, 128, 64), (256, 128, 63), (256, 64, 64), (127, 128, 64), (64, 128, 64), (-256, 128, 64)):
        refused(lambda: CALLS["read"](c, n=2, strides=strides), "overlap")
    refused(lambda: moert.check(moert.lib().moert_kv8_append(c._p, 0, 1, None, None, 1, None)), "null rows")


def test_bad_attentions_are_refused():
    c = cache()
    for heads in (0, -2, 3, 130):
        refused(lambda: CALLS["attend"](c, heads=heads), "query heads")
        refused(lambda: c.workspace(heads), "query heads")
    for n in (0, -1, 97):
        refused(lambda: CALLS["attend"](c, n=n), "positions")
        refused(lambda: c.workspace(4, n), "positions")
    for scale in (math.nan, math.inf, -math.inf):
        refused(lambda: CALLS["attend"](c, scale=scale), "scale")
    for decay in (math.nan, 1.5, math.inf):
        refused(lambda: CALLS["attend"](c, mass_decay=decay), "mass_decay")
    refused(lambda: CALLS["attend"](cache({"mass": None}), mass_decay=1.0), "null buffer")
    refused(lambda: CALLS["attend"](c, q=None), "null rows")
    refused(lambda: CALLS["attend"](c, out=None), "null rows")
    refused(lambda: CALLS["attend"](c, out_strides=(256, 256, 0)), "overlap")
    refused(lambda: CALLS["attend"](c, ws=None), "workspace")
    refused(lambda: CALLS["attend"](c, ws=0x30008), "workspace")
    for track in (False, True):
        need = c.workspace(4, 3, track=track)
        assert need > 0
        refused(lambda: CALLS["attend"](c, n=3, mass_decay=1.0 if track else None, ws_bytes=need - 1), "workspace")
    rows = c._rows(0x20000, moert.F32, None, 1, 4)
    half = c._rows(0x20000, moert.F16, None, 1, 4)
    refused(lambda: moert.check(moert.lib().moert_kv8_attend(
        c._p, 0, 2, 4, 1, 0.125, rows, half, -1.0, 0x30000, 1 << 30, None)), "dtype")
    big = cache(seqs=65535, max_len=1 << 20)
    refused(lambda: big.workspace(64, 1 << 12), "sequences")
    with pytest.raises(moert.MoertError):
        moert.check(moert.lib().moert_kv8_workspace(c._p, 2, 4, 1, 0, None))


def test_bad_evictions_are_refused():
    for bad in (dict(keep=-1), dict(keep=2, first=-1), dict(keep=2, last=-1), dict(keep=2, first=3),
                dict(keep=2, first=1, last=2), dict(keep=2 ** 31 - 1, first=2 ** 31 - 1, last=2 ** 31 - 1)):
        refused(lambda: CALLS["evict"](cache(), **bad), "keep")
    refused(lambda: CALLS["evict"](cache({"mass": None})), "null buffer")
    c = cache()
    refused(lambda: moert.check(moert.lib().moert_kv8_lengths(c._p, 0, 1, None, None)), "null lengths")


@pytest.mark.parametrize("d", [64, 128])
def test_shapes_and_the_order_of_v(d):
    shapes = moert.kv8_shapes(3, 2, d, 320)
    assert shapes["k_codes"] == ((3, 2, 10, 32, d), np.uint8) and shapes["state"] == ((3, 4), np.int32)
    assert {n + "_dev" for n in shapes} == {n for n, _ in moert.moert_kv8._fields_[4:]}
    places = ku.v_order(d)
    assert sorted(places.reshape(-1).tolist()) == list(range(32 * d))
    # the eight positions of an element that one lane multiplies lie side by side
    for e in (0, 1, d - 1):
        for g in range(4):
            t = [4 * g + j for j in range(4)] + [16 + 4 * g + j for j in range(4)]
            assert np.array_equal(np.diff(places[t, e]), np.ones(7))


def test_the_definition_does_not_depend_on_how_rows_are_appended():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 1, 150, 2, 64)).astype(np.float32)
    a, b = ku.Cache(1, 2, 64, 160), ku.Cache(1, 2, 64, 160)
    a.append(k, v)
    for i in (0, 1, 33, 64, 95, 149):
        j = {0: 1, 1: 33, 33: 64, 64: 95, 95: 149, 149: 150}[i]
        b.append(k[:, i:j], v[:, i:j])
    assert a.len(0) == b.len(0) == 150
    for h in range(2):
        for x, y in zip(a.rows(0, h), b.rows(0, h)):
            assert np.array_equal(x, y)
    got, _, _ = a.rows(0, 0)
    want = k[0, :, 0].astype(np.float64)
    # half a step of the code, 1 / 254 of the block's largest magnitude, and the rounding to fp16
    assert np.abs(got - want).max() <= np.abs(want).max() * (1 / 254 + 2.0 ** -11) * (1 + 2.0 ** -20)


def test_the_definition_of_poison_and_zero_blocks():
    x = np.zeros((32, 64), np.float16)
    assert ku.code_block(x)[1] == 1.0
    x[3, 5] = 127.0
    codes, s = ku.code_block(x)
    assert s == 1.0 and codes[3, 5] == 127
    x[4, 6] = 0.5  # a tie: to even
    x[4, 7] = 1.5
    codes, _ = ku.code_block(x)
    assert codes[4, 6] == 0 and codes[4, 7] == 2
    x[0, 0] = np.inf
    assert np.isnan(ku.code_block(x)[1])


def test_the_definition_of_evictions():
    c = ku.Cache(1, 1, 64, 320)
    rows = np.random.default_rng(2).standard_normal((1, 263, 1, 64))
    c.append(rows, rows)
    for b, m in enumerate([5.0, 1.0, 1.0, 0.0, np.nan, 1.0, 0.0, 9.0]):
        c.blocks[0][0][b][4] = m
    kept = [id(x) for x in c.blocks[0][0]]
    c.evict(5, 1, 1)  # blocks 0 and 7 stay; of 1 .. 6: NaN first, then 1, 1 (the earlier ones)
    assert [kept.index(id(x)) for x in c.blocks[0][0]] == [0, 1, 2, 4, 7]
    assert c.len(0) == 5 * 32 + 7
    c.evict(9, 0, 0)
    assert c.len(0) == 5 * 32 + 7


def test_a_workspace_does_for_every_smaller_attention():
    rng = np.random.default_rng(6)
    for _ in range(300):
        seqs, kv_heads, group = int(rng.integers(1, 40)), int(rng.integers(1, 9)), int(rng.integers(1, 9))
        c = cache(seqs=seqs, kv_heads=kv_heads, head_dim=int(rng.choice([64, 128])),
                  max_len=32 * int(2 ** rng.uniform(0, 12)))
        n = int(rng.integers(1, c.max_len + 1))
        a, b = int(rng.integers(1, seqs + 1)), int(rng.integers(1, n + 1))
        heads = kv_heads * group
        for track in (False, True):
            assert c.workspace(heads, b, n_seqs=a, track=track) <= c.workspace(heads, n, n_seqs=seqs, track=track)
            assert c.workspace(heads, b, n_seqs=a) <= c.workspace(heads, b, n_seqs=a, track=True)
