"""Attention over the paged K/V cache in every kernel that a call may choose (tests/pages_forms.py), against the definition
in 64 bits."""
import numpy as np
import pytest

import moert
import pages_forms as pf
import pages_util as pu
from test_gpu_pages import both, cache_type, hip, normal, queries, step  # noqa: F401 (hip: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(pf.TYPES))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("name", [n for n in pf.FORMS if "streamed" not in n])
def test_forms(hip, name, d, dtype):  # noqa: F811
    rng = np.random.default_rng(61)
    call, (seqs, H, page, pages, max_pages), heads, before, new, _ = pf.FORMS[name]
    dev, ref = both(hip, seqs, H, d, page, pages, max_pages, dtype=cache_type(dtype))
    step(dev, ref, rng, before, dtype)
    starts = step(dev, ref, rng, new, dtype)
    q, x = queries(rng, dtype, sum(new), heads, d)
    pu.check(getattr(dev, call)(q, d ** -0.5, dtype, starts=starts), ref.attend(x, starts, d ** -0.5, dtype), dtype)


@pytest.mark.parametrize("dtype", list(pf.TYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_a_cache_that_is_streamed(hip, d, dtype):  # noqa: F811
    """A pool of more than the last-level cache keeps of a few layers: its pages anywhere, most of it never written."""
    rng = np.random.default_rng(63)
    call, (seqs, H, page, pages, max_pages), heads, before, new, _ = pf.FORMS["positions, streamed"]
    dev = pu.Device(hip, seqs, H, d, page, pages, max_pages, dtype=cache_type(dtype))
    ref = pu.Cache(seqs, H, d, page, 4, max_pages, dtype=cache_type(dtype))
    high, lens = np.array([199, 3, 150, 77]), [a + b for a, b in zip(before, new)]
    ref.table, ref.rows, at = [[0, 1, 2], [3]], lens, np.concatenate([np.arange(lens[0]), 3 * page + np.arange(lens[1])])
    k, v = (pu.to_bits(normal(rng, len(at), H, d), dtype) for _ in range(2))
    dev.append(k, v, high[at // page] * page + at % page, dtype)
    ref.append(k, v, at, dtype)
    table = np.full((seqs, max_pages), -1)
    table[0, :3], table[1, 0] = high[:3], high[3]
    dev.set("table", table)
    dev.set("state", [[n, 0, n - 1, 0] for n in lens])
    q, x = queries(rng, dtype, 3, heads, d)
    pu.check(dev.attend(q[:2], d ** -0.5, dtype), ref.attend(x[:2], [0, 1, 2], d ** -0.5, dtype), dtype)
    starts = [0, 0, 1]  # one that is idle, and rows behind the last
    pu.check(dev.attend(q, d ** -0.5, dtype, starts=starts), ref.attend(x, starts, d ** -0.5, dtype), dtype)


@pytest.mark.parametrize("dtype", list(pf.TYPES))
@pytest.mark.parametrize("d", [64, 128])
def test_attentions_of_a_part_of_the_sequences(hip, d, dtype):  # noqa: F811
    """Calls for some sequences that follow each other, from the first's table, state and starts on, each with a workspace of
    its own: the others' rows stay as they were, and the parts together do what one call for all does."""
    rng = np.random.default_rng(65)
    S, H, heads, page, max_pages = 7, 2, 6, 32, 60
    dev, ref = both(hip, S, H, d, page, 120, max_pages, dtype=cache_type(dtype))
    step(dev, ref, rng, [500, 40, 0, 33, 1000, 7, 64], dtype)
    new = [1, 70, 1, 300, 1, 0, 1]
    starts = step(dev, ref, rng, new, dtype, tokens=sum(new) + 4)
    tokens = sum(new) + 4
    q, x = queries(rng, dtype, tokens, heads, d)
    at = hip.upload(starts)
    qp = hip.upload(q)

    def part(s0, n):
        buffers = dict(dev.at, table=dev.at["table"] + 4 * s0 * max_pages, state=dev.at["state"] + 16 * s0)
        c = moert.Pages(n, H, d, page, 120, max_pages, buffers, dtype=cache_type(dtype))
        size = c.workspace(heads, tokens)
        return c, dict(starts=at + 4 * s0, tokens=tokens, ws=hip.upload(np.full(max(size, 16), 0xFF, np.uint8)), ws_bytes=size,
                       dtype=dtype)

    long, off, _ = ref.attend(x, starts, d ** -0.5, dtype, which=lambda m: m >= 2)
    for s0, n in ((1, 1), (3, 3), (0, 2), (2, 5)):
        c, kw = part(s0, n)
        out = dev._out(q, dtype)
        c.prompt(qp, out, heads, d ** -0.5, least=2, **kw)
        hip.sync()
        wrote = np.zeros(tokens, bool)
        for s in range(s0, s0 + n):
            wrote[starts[s]:starts[s + 1]] = new[s] >= 2
        pu.check(hip.get(out, q.shape, q.dtype), (long, off, wrote), dtype)
    out = dev._out(q, dtype)
    for call, s0, n in (("prompt", 0, 2), ("prompt", 2, 5), ("attend", 0, 3), ("attend", 3, 4)):
        c, kw = part(s0, n)
        getattr(c, call)(qp, out, heads, d ** -0.5, **kw, **(dict(least=2) if call == "prompt" else {}))
    hip.sync()
    pu.check(hip.get(out, q.shape, q.dtype), ref.attend(x, starts, d ** -0.5, dtype), dtype)
