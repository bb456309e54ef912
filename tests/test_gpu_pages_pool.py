"""What an append to the paged K/V cache leaves in the pool, slot by slot, also where it is neither a row nor nothing."""
import numpy as np
import pytest

import pages_util as pu
from pages_util import BF16, F16, F32
from test_gpu_pages import both, cache_type, hip, normal  # noqa: F401 (hip: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [150, 3000])
def test_poisoned_rows_are_written_and_others_left(hip, dtype, d, rows):  # noqa: F811
    """A row that is not finite becomes a K of NaN and a V of exactly 0, in one KV head, whether its run of positions leaves
    together or not; a finite row lies beside it bit for bit, and a slot that no row names is as it was, in every bit. Of few
    and of many rows: a workgroup takes 8 or 32."""
    rng = np.random.default_rng(rows + d)
    H, page = 3, 64
    dev, ref = both(hip, 1, H, d, page, 70, 70, dtype=cache_type(dtype))
    slots = np.arange(5, 5 + rows)
    slots[rows // 2:] = 5 + rows // 2 + rng.permutation(rows - rows // 2)  # runs in order, then none
    slots[rng.random(rows) < 0.15] = -1
    k, v = normal(rng, rows, H, d), normal(rng, rows, H, d)
    for x in (k, v):
        x[rng.random((rows, H)) < 0.05, rng.integers(d)] = rng.choice([np.inf, -np.inf, np.nan])
    k, v = pu.to_bits(k, dtype), pu.to_bits(v, dtype)
    dev.append(k, v, slots, dtype)
    ref.append(k, v, slots, dtype)
    written = np.zeros(70 * page, bool)
    written[slots[slots >= 0]] = True
    bad = np.isnan(ref.k).any(2) & written[:, None]
    fine = ~bad & written[:, None]
    assert bad.any() and fine.any() and not written.all() and np.array_equal(bad, np.isnan(ref.v).any(2) & written[:, None])
    t, e = np.arange(pu.B)[:, None], np.arange(d)[None, :]
    for name, place, want in (("k", pu.k_place(t, e), ref.k), ("v", pu.v_place(t, e, d), ref.v)):
        got = dev.array(name)[..., place].transpose(0, 2, 3, 1, 4).reshape(want.shape)
        assert (got[~written] == 0xFFFF).all(), name
        assert np.array_equal(got[fine], pu.to_bits(want.astype(np.float32), ref.dtype)[fine]), name
        if name == "k":
            assert ((got[bad] & 0x7FFF) > pu.INF[ref.dtype]).all() and (got[bad] != 0xFFFF).all()
        else:
            assert not got[bad].any()
