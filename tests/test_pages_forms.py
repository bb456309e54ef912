"""Which kernels, down to their variants, the attentions of pages_forms.py launch: without a device."""
import pytest

import moert
import pages_forms as pf
from test_pages_launches import launches  # noqa: F401 (a fixture)


@pytest.mark.parametrize("d", [64, 128])
def test_forms_take_their_kernels(launches, d):  # noqa: F811
    cases, want = [], []
    for name, (call, (seqs, H, page, pages, max_pages), heads, before, new, kernels) in pf.FORMS.items():
        for dtype in pf.TYPES:
            cases.append(dict(call=call, cache=(seqs, H, d, page, pages, max_pages),
                              dtype=moert.BF16 if dtype == moert.BF16 else moert.F16,
                              kw=dict(heads=heads, tokens=sum(new), dtype=dtype)))
            want.append((name, [pf.kernel(k, d, dtype) for k in kernels]))
    for (name, names), got in zip(want, launches(cases)):
        assert got[0] == 0 and len(got[1]) == len(names), (name, got)
        assert all(n in line[0] for n, line in zip(names, got[1])), (name, got)


def test_every_kernel_of_an_attention_is_in_a_form():
    taken = {pf.kernel(k, d, dtype) for *_, kernels in pf.FORMS.values() for k in kernels for d in (64, 128) for dtype in pf.TYPES}
    assert len(taken) == 6 * (2 + 1 + 4)


def test_a_part_of_the_sequences_takes_kernels_of_its_own(launches):  # noqa: F811
    """A prompt of 900 rows beside 63 single rows: tiles of 16 rows in a call for all sequences, of 128 in one for its own."""
    whole, part = (dict(call="prompt", cache=(seqs, 8, 64, 64, 500, 100), kw=dict(heads=24, tokens=963, least=2)) for seqs in (64, 1))
    got = launches([whole, part])
    assert "k_pages_cols" in got[0][1][0][0] and "k_pages_tiles" in got[1][1][0][0]
