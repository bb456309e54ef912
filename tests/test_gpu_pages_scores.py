"""Attention over the paged K/V cache where its scores are hardest: large ones a few steps of f32 apart, factors beyond
f32's exponents, weights whose rounding shows. Bounds follow from the roundings that include/moert.h states."""
import numpy as np
import pytest

import pages_util as pu
from pages_util import BF16, F16, F32
from test_gpu_pages import both_ways, cache_type, hip, normal, one_sequence  # noqa: F401 (hip: a fixture)

pytestmark = pytest.mark.gpu

TWO = {F32: 2.0 ** -21, F16: 2.0 ** -21, BF16: 2.0 ** -15}  # weights as two numbers of the cache's type, and their sum


def weight_error(dtype, m):
    """Of a weight, relative: as two numbers (one position), or rounded once and its sum with it (prompts)."""
    return TWO[dtype] if m == 1 or dtype == F32 else 2 * pu.HALF[dtype]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("first", [0, 200])
def test_large_scores_a_few_steps_apart(hip, dtype, d, sign, first):  # noqa: F811
    """Four rows of about 2^24 as sums of products, 0 to 9 steps of f32 apart, in blocks that one wave takes one after the
    other, times factors that make scores of 2^16 to 2^44 and of 10^35 of them, many of them where one step is about what
    moves a maximum; the others are far below. Their differences are exact, and so the weights differ by little more than
    their roundings: of the factor and the exponent, 2^-22 of an exponent below 32 (a smaller weight is below 2^-24), of
    exp2, of sums, and of what the second product takes. From row 200 on the prompts' waves have been through stages of
    small scores before."""
    rng = np.random.default_rng(51)
    rows, n, heads = first + 3 * 128 + 40, 7, 4
    at = first + 128 * np.arange(4)
    v = normal(rng, rows, 1, d)
    few = [m * 2.0 ** e for e in range(-8, 20) for m in (1.0, 1.37)] + [1e27, 1.1e28]
    many = [(1 + m / 64) * 2.0 ** e for e in range(9) for m in range(64)]
    for step, order, scales in ((1, (0, 1, 2, 3), many), (3, (0, 1, 2, 3), few), (1, (1, 0, 3, 2), few)):
        q, k = np.zeros((n, heads, d), np.float32), np.zeros((rows, 1, d), np.float32)
        q[..., 0], q[..., 1] = sign * 4080.0, step
        k[:, 0, 0] = 0.0 if sign > 0 else 4096.0
        k[at, 0, 0], k[at, 0, 1] = 4080.0, order
        b = pu.to_bits(q, dtype)
        dev, ref = one_sequence(hip, dtype, k, v)
        x = ref.kv(0, 0, rows)[1][at]
        for scale in np.float32(scales).tolist():
            s = scale * step * np.array(order, np.float64)
            p = np.exp(s - s.max())
            p /= p.sum()
            want = p @ x
            for m, out in both_ways(dev, b, scale, dtype):
                off = (2.0 ** -16 + weight_error(dtype, m)) * (p @ np.abs(x)) + 2.0 ** -20 * np.abs(x).max() + \
                    pu.HALF[dtype] * np.abs(want)
                err = np.abs(pu.from_bits(out, dtype) - want)
                assert (err <= off).all(), (scale, step, order, m, (err / off).max())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [0.0, 1e-45, 1e-40, -1e-39, 3e-39, -1e-38])
def test_scales_without_a_normal_factor(hip, dtype, d, scale):  # noqa: F811
    """Scales of 0 and of f32's smallest, beside the largest products that the type lets through (bf16: of 10^38): the
    products of scale 0 all weigh the same."""
    rng = np.random.default_rng(53)
    rows, n = 333, 7
    big = {F32: (1e38 / 60000.0 / d, 60000.0), F16: (60000.0, 60000.0), BF16: (2.0 ** 60, 1e38 / 2.0 ** 60 / d)}[dtype]
    q = np.full((n, 4, d), big[0], np.float32)
    k = (rng.choice([-1.0, -0.5, 0.0, 0.5, 1.0], (rows, 1, 1)) * big[1] * 0.99 * np.ones(d)).astype(np.float32)
    dev, ref = one_sequence(hip, dtype, k, normal(rng, rows, 1, d))
    b = pu.to_bits(q, dtype)
    scale = float(np.float32(scale))
    for m, out in both_ways(dev, b, scale, dtype):
        pu.check(out, ref.attend(pu.from_bits(b[-m:], dtype), [0, m], scale, dtype), dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("max_pages", [7, 256])
def test_one_positions_weights_are_two_numbers(hip, dtype, d, max_pages):  # noqa: F811
    """Half of the rows weigh 1, half exp(-s), s of 1/16 to 4; their V cancel for one element of each head, so that an
    output's own rounding does not hide a weight's, which has one sign in all rows. Scores are exact; the factor, the
    exponent, exp2 and sums bring 2^-19 at most (of exponents below 13 their f32 roundings, 2^-20)."""
    rows, heads = 400, 64
    s = (1 + np.arange(heads)) / 16
    k, v = np.zeros((rows, 1, d), np.float32), np.ones((rows, 1, d), np.float32)
    k[1::2, 0, 0] = -1.0
    cancel = pu.from_bits(pu.to_bits(np.exp(s[np.arange(d) % heads]), cache_type(dtype)), cache_type(dtype))
    v[1::2, 0] = -cancel
    dev, ref = one_sequence(hip, dtype, k, v, max_pages)
    q = np.zeros((1, heads, d), np.float32)
    q[..., 0] = s
    w = np.exp(-s)[:, None]
    want = (1 - w * cancel) / (1 + w)
    size = (1 + w * cancel) / (1 + w)
    off = (2.0 ** -19 + TWO[dtype]) * size + pu.HALF[dtype] * np.abs(want) + (2.0 ** -24 if dtype == F16 else 0.0)
    once = pu.from_bits(pu.to_bits(w, cache_type(dtype)), cache_type(dtype))
    assert (np.abs((1 - once * cancel) / (1 + w) - want) > 4 * off).any()  # weights rounded once would show
    err = np.abs(pu.from_bits(dev.attend(pu.to_bits(q, dtype), 1.0, dtype), dtype)[0] - want)
    assert (err <= off).all(), (err / off).max()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_many_small_weights(hip, dtype, d):  # noqa: F811
    """20000 rows of 2^-18 to 2^-24 of the largest weight, as 16-bit numbers below fp16's normal ones: all V are 1, and so is
    the output, as long as sums and products hold the same weights. What a weight below fp16's steps (2^-31 of the largest)
    loses is 2^-17 of the output at most, in one of the two."""
    rows, n = 20000, 7
    k = np.zeros((rows, 1, d), np.float32)
    k[1:, 0, 0] = -1.0
    dev, ref = one_sequence(hip, dtype, k, np.ones((rows, 1, d)))
    for power in (18.0, 20.5, 21.25, 22.0, 24.0):
        q = np.zeros((n, 4, d), np.float32)
        q[..., 0] = power
        for m, out in both_ways(dev, pu.to_bits(q, dtype), float(np.float32(np.log(2))), dtype):
            err = np.abs(pu.from_bits(out, dtype) - 1.0)
            assert (err <= pu.HALF[dtype] + 2.0 ** -16).all(), (power, m, err.max())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["subnormal", "large", "falling", "rising", "equal"])
def test_extremes_of_wide_heads(hip, dtype, kind):  # noqa: F811
    """Heads of 128: values at the ends of their types, scores that fall or rise all along by up to 900, and equal ones of
    10^9, in caches that are split and not."""
    rng = np.random.default_rng(55)
    rows, n, d = 700, 7, 128
    k, v, q, scale = normal(rng, rows, 1, d), normal(rng, rows, 1, d), normal(rng, n, 4, d), 0.0625
    if kind == "subnormal":
        k, v, q, scale = k * 3e-6, v * 3e-6, q * 3e-6, 1e10
    elif kind == "large":
        k, v = np.clip(k, -1, 1) * 60000, np.clip(v * 4, -1, 1) * 65504
        q, scale = q * 1e3, 1e-8
    elif kind in ("falling", "rising"):
        k = np.broadcast_to(np.linspace(0, 7, rows)[:, None, None], k.shape)
        k = k[::-1] if kind == "falling" else k
        q, scale = np.ones_like(q), 1.0
    else:
        k, q, scale = np.full_like(k, 300.0), np.full_like(q, 500.0), 52.0
    for max_pages in (11, 256):
        dev, ref = one_sequence(hip, dtype, k, v, max_pages)
        b = pu.to_bits(q, dtype)
        for m, out in both_ways(dev, b, scale, dtype):
            want = ref.attend(pu.from_bits(b[-m:], dtype), [0, m], 0.0 if kind == "equal" else scale, dtype)
            pu.check(out, want, dtype)


@pytest.mark.parametrize("power", [4, 8, 12, 16, 20])
def test_small_elements_of_f32_queries(hip, power):  # noqa: F811
    """All of a score comes from an element of 2^-power of its row's largest, which meets zeros: as two fp16 it is off by
    2^-22 of itself, or by 2^-34 of the largest. A weight is off by the factor of its own score's and of the sum's; exp2,
    the factor, exponents below 16 and sums bring 2^-18."""
    rng = np.random.default_rng(57)
    rows, n, d = 300, 7, 64
    x = 1.37 * 2.0 ** -power
    scale = float(np.float32(4.0 / (60000.0 * x)))
    k = np.zeros((rows, 1, d), np.float32)
    k[..., 1] = rng.uniform(-60000, 60000, (rows, 1))
    dev, ref = one_sequence(hip, F32, k, normal(rng, rows, 1, d))
    q = np.zeros((n, 4, d), np.float32)
    q[..., 0], q[..., 1] = 1.0, x
    off = 2 * scale * 60000.0 * (2.0 ** -22 * x + 2.0 ** -34) + 2.0 ** -18 + TWO[F32]
    for m, out in both_ways(dev, q, scale, F32):
        for i in range(m):
            kk, vv = ref.kv(0, 0, rows - m + 1 + i)
            s = scale * np.float64(np.float32(x)) * kk[:, 1]
            p = np.exp(s - s.max())
            p /= p.sum()
            err = np.abs(out[i] - p @ vv)
            assert (err <= off * (p @ np.abs(vv)) + 2.0 ** -24 * np.abs(vv).max()).all(), (m, i, err.max())
