"""The paged K/V cache without a device: every refusal comes before anything is launched, the buffers' shapes, the layout
of a block, and the definition that the GPU tests compare with (tests/pages_util.py) against plain facts."""
import math

import numpy as np
import pytest

import moert
import pages_util as pu
from pages_util import BF16, F16, F32

GOOD = dict(seqs=2, kv_heads=2, head_dim=64, page=64, pages=10, max_pages=4, dtype=F16)


def cache(buffers=None, **kw):
    at = {n[:-4]: 0x10000 for n, _ in moert.moert_pages._fields_[7:]}  # never reached
    at.update(buffers or {})
    return moert.Pages(**{**GOOD, **kw}, buffers=at)


CALLS = {
    "clear": lambda c, **kw: c.clear(**kw),
    "plan": lambda c, **kw: c.plan(**{**dict(new=0x20000, tokens=3, starts=0x30000, slots=0x40000,
                                             positions=0x50000), **kw}),
    "append": lambda c, **kw: c.append(**{**dict(k=0x20000, v=0x20000, slots=0x30000, tokens=1), **kw}),
    "workspace": lambda c, **kw: c.workspace(**{**dict(heads=4), **kw}),
    "attend": lambda c, **kw: c.attend(**{**dict(q=0x20000, out=0x20000, heads=4, scale=0.125, ws=0x30000,
                                                 ws_bytes=1 << 40), **kw}),
    "prompt": lambda c, **kw: c.prompt(**{**dict(q=0x20000, out=0x20000, heads=4, scale=0.125, starts=0x30000,
                                                 tokens=5, ws=0x40000, ws_bytes=1 << 40), **kw}),
    "lengths": lambda c, **kw: c.lengths(**kw),
}
USES = {"clear": "free state", "plan": "free state table", "append": "state k v", "workspace": "state",
        "attend": "state k v table", "prompt": "state k v table", "lengths": "state"}


def refused(call, what):
    with pytest.raises(moert.MoertError) as e:
        call()
    assert e.value.code == moert.E_CONFIG, e.value
    assert what in str(e.value), e.value


@pytest.mark.parametrize("name", sorted(CALLS))
def test_bad_caches_are_refused(name):
    call = CALLS[name]
    for bad in (dict(seqs=0), dict(seqs=65536), dict(kv_heads=0), dict(kv_heads=257), dict(seqs=8192, kv_heads=129),
                dict(head_dim=32), dict(head_dim=96), dict(page=16), dict(page=0), dict(page=96), dict(page=512),
                dict(pages=0), dict(pages=(1 << 24) + 1), dict(pages=1 << 24, kv_heads=33), dict(max_pages=0),
                dict(max_pages=(1 << 14) + 1), dict(seqs=65535, kv_heads=1, max_pages=1 << 14 + 1, page=32),
                dict(dtype=F32), dict(dtype=1), dict(dtype=5), dict(dtype=-1)):
        refused(lambda: call(cache(**bad)), "pages_" + name)
    for buf in USES[name].split():
        refused(lambda: call(cache({buf: None})), "null buffer")
        refused(lambda: call(cache({buf: 0x10002})), "aligned")


@pytest.mark.parametrize("name", sorted(set(CALLS) - {"workspace"}))
def test_a_cache_that_is_not_device_memory_is_refused(name):
    host = np.zeros(1 << 16, np.uint8)
    at = host.ctypes.data + -host.ctypes.data % 16
    refused(lambda: CALLS[name](cache({n[:-4]: at for n, _ in moert.moert_pages._fields_[7:]})), "not in device memory")


def test_a_null_cache_and_unknown_buffers_are_refused():
    assert moert.lib().moert_pages_clear(None, None) == moert.E_CONFIG
    with pytest.raises(ValueError):
        cache({"keys": 1})
    assert moert.lib().moert_pages_workspace(cache()._p, 4, 0, None) == moert.E_CONFIG


def test_bad_arrays_and_rows_are_refused():
    c = cache()
    for name in ("plan", "append", "attend", "prompt", "workspace"):
        for n in (-1, (1 << 24) + 1):
            refused(lambda: CALLS[name](c, tokens=n), "rows")
    for bad in (dict(new=0), dict(new=0x20001), dict(starts=0), dict(starts=0x20002), dict(slots=0), dict(slots=0x20003),
                dict(positions=0x20002)):
        refused(lambda: CALLS["plan"](c, **bad), "array")
    for bad in (dict(slots=0), dict(slots=0x20002)):
        refused(lambda: CALLS["append"](c, **bad), "array")
    for bad in (dict(starts=0), dict(starts=0x20002)):
        refused(lambda: CALLS["prompt"](c, **bad), "array")
    refused(lambda: CALLS["attend"](c, starts=0x20002), "array")
    for name, rows in (("append", ("k", "v")), ("attend", ("q", "out")), ("prompt", ("q", "out"))):
        for r in rows:
            refused(lambda: CALLS[name](c, **{r: None}), "null rows")
            refused(lambda: CALLS[name](c, dtype=F32, **{r: 0x20002}), "not aligned")
            refused(lambda: CALLS[name](c, **{r: 0x20001}), "not aligned")
        for dtype in (moert.Q8_0, moert.Q4_0, BF16, 5, -1):
            refused(lambda: CALLS[name](c, dtype=dtype), "dtype")
        for dtype in (F32, F16):
            refused(lambda: CALLS[name](cache(dtype=BF16), dtype=dtype), "dtype")


def test_bad_attentions_are_refused():
    c = cache()
    for name in ("attend", "prompt"):
        for heads in (0, -2, 1, 3, 130):
            refused(lambda: CALLS[name](c, heads=heads), "heads")
        for scale in (math.inf, -math.inf, math.nan):
            refused(lambda: CALLS[name](c, scale=scale), "scale")
        kw = dict(tokens=3, starts=0x30000)
        for strides in ((255, 64), (256, 63), (0, 64), (64, 64), (-256, 64)):
            refused(lambda: CALLS[name](c, out_strides=strides, **kw), "overlap")
    for heads in (0, 3, 130):
        refused(lambda: CALLS["workspace"](c, heads=heads), "heads")
    refused(lambda: CALLS["attend"](c, tokens=1), "without starts")
    refused(lambda: CALLS["attend"](c, tokens=3), "without starts")
    for least in (0, -1):
        refused(lambda: CALLS["prompt"](c, least=least), "at least")
    refused(lambda: CALLS["prompt"](c, tokens=1 << 24, heads=16), "rows")
    refused(lambda: CALLS["attend"](cache(seqs=65535, kv_heads=8, max_pages=1), tokens=5, starts=0x30000, heads=512),
            "heads")
    for seqs in ((-1, 1), (2, 1), (0, 3), (0, 0), (1, -1)):
        refused(lambda: c.lengths(*seqs), "sequences")


def test_workspaces():
    """A workspace that is too small or not aligned is refused; none is needed where sequences are never split."""
    for kw in (dict(max_pages=4096, pages=5000, seqs=1), dict(max_pages=64, seqs=4)):
        c = cache(**kw)
        size = c.workspace(4)
        assert size > 0
        refused(lambda: CALLS["attend"](c, ws_bytes=size - 1), "workspace")
        refused(lambda: CALLS["attend"](c, ws=0x30008, ws_bytes=size), "workspace")
        refused(lambda: CALLS["attend"](c, ws=0, ws_bytes=size), "workspace")
    assert cache(max_pages=1).workspace(4) == 0


def test_no_rows_need_nothing():
    c = cache()
    CALLS["append"](c, tokens=0, slots=0)
    CALLS["prompt"](c, tokens=0)
    CALLS["attend"](c, tokens=0, starts=0x30000)


def test_shapes_and_layout():
    s = moert.pages_shapes(3, 2, 64, 128, 10, 5)
    assert s["k"] == s["v"] == ((10, 2, 4, 2048), np.uint16)
    assert s["table"] == ((3, 5), np.int32) and s["state"] == ((3, 4), np.int32) and s["free"] == ((11,), np.int32)
    for d in (64, 128):
        t, e = np.arange(32)[:, None], np.arange(d)[None, :]
        for place in (pu.k_place(t, e), pu.v_place(t, e, d)):
            assert sorted(place.reshape(-1).tolist()) == list(range(32 * d))
        assert pu.v_place(21, 3, d) - pu.v_place(20, 3, d) == 1 and pu.v_place(24, 3, d) - pu.v_place(16, 3, d) == 4
        assert pu.k_place(4, 8) - pu.k_place(3, 8) == 8


def test_definition_plans():
    c = pu.Cache(3, 1, 64, 32, 4, 3)
    starts, slots, pos = c.plan([33, 1, 64], 100)
    assert starts.tolist() == [0, 33, 34, 98] and c.table == [[0, 1], [2], []]  # two pages for the last, one is left
    assert slots.tolist() == list(range(33)) + [64] + [-1] * 66 and pos.tolist() == list(range(33)) + [0] + [-1] * 66
    assert c.refused == [0, 0, 64] and c.first == [0, 0, -1] and c.seen(2) == 0 and c.free == [3]
    starts, slots, pos = c.plan([-1, 32, 64], 96)
    assert c.table == [[], [2, 1], [0, 3]] and starts.tolist() == [0, 0, 32, 96]
    assert slots[:32].tolist() == list(range(65, 96)) + [32] and slots[32:].tolist() == list(range(32)) + list(range(96, 128))
    assert c.rows == [0, 33, 64] and c.refused == [0, 0, 64] and c.first == [0, 1, 0]


def test_definition_attends():
    rng = np.random.default_rng(0)
    c = pu.Cache(1, 1, 64, 32, 4, 4)
    _, slots, _ = c.plan([40], 40)
    k, v = (pu.to_bits(rng.standard_normal((40, 1, 64)).astype(np.float32), F16) for _ in range(2))
    c.append(k, v, slots, F16)
    q = rng.standard_normal((40, 2, 64))
    out, off, wrote = c.attend(q, [0, 40], 0.125, F32)
    kk, vv = pu.from_bits(k, F16)[:, 0], pu.from_bits(v, F16)[:, 0]
    for i in (0, 7, 39):
        w = np.exp(0.125 * kk[:i + 1] @ q[i, 1])
        assert np.allclose(out[i, 1], w @ vv[:i + 1] / w.sum(), rtol=1e-12)
    assert wrote.all() and (off > 0).all() and (off < 1e-3).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_roundings(dtype):
    x = np.array([1.0, 1 + pu.HALF[dtype], 1 + 3 * pu.HALF[dtype], -2.5, 0.0, np.inf, np.nan], np.float32)
    got = pu.from_bits(pu.to_bits(x, dtype), dtype)
    step = 2 * pu.HALF[dtype]
    assert got[:5].tolist() == [1.0, 1.0, 1 + 2 * step, -2.5, 0.0] and np.isinf(got[5]) and np.isnan(got[6])
