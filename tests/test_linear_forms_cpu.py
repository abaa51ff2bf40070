"""The cases of tests/linear_forms.py lead to the kernels that they are for (no GPU: pb_linear_form answers on the host)."""
import random

import pytest

import linear_forms as forms
from pixelbox_amd import capi


@pytest.mark.parametrize("kind,align,m,groups,n,k,form", forms.CASES)
def test_the_case_takes_its_form(kind, align, m, groups, n, k, form):
    assert capi.linear_form(forms.TYPE[kind], m, n, k, groups, align) == form
    ld = forms.row_stride(kind, k, align) * forms.SIZE[kind]
    assert ld % align == 0 and (align == 16 or ld % (2 * align) != 0)


@pytest.mark.parametrize("kind", list(forms.ALIGN))
def test_no_tile_form_of_a_grouped_product_is_left_out(kind):
    rng = random.Random(kind)
    for align in forms.ALIGN[kind]:
        listed = {(c[6], c[3] > 64) for c in forms.CASES if c[:2] == (kind, align)}
        for _ in range(4000):
            m, n, k = (int(2 ** rng.uniform(a, b)) for a, b in ((5, 13), (5, 13), (5, 12)))
            groups = rng.choice((2, 3, 5, 8, 17, 33, 64, 66, 100, 200))
            if m < 2 * groups or m * n * k > 1 << 37:
                continue
            form = capi.linear_form(forms.TYPE[kind], m, n, k, groups, align)
            assert form < 3 or (form, True) in listed, (kind, align, m, n, k, groups, form)
            assert form < 3 or (form, False) in listed, (kind, align, m, n, k, groups, form)


def test_refusals_of_the_form_query():
    ok = dict(type_=0, m=5, n=5, k=5, groups=0, align=16)
    assert 0 <= capi.linear_form(**ok) <= 6
    for change in (dict(type_=4), dict(type_=-1), dict(m=0), dict(m=1 << 31), dict(n=0), dict(n=1 << 31), dict(k=(1 << 28) + 1), dict(groups=1025), dict(align=0),
                   dict(align=3), dict(align=32), dict(m=(1 << 31) - 257, n=1 << 29)):
        with pytest.raises(capi.PixelboxError) as e:
            capi.linear_form(**{**ok, **change})
        assert e.value.code == -1 and "pb_linear_form" in str(e.value), change
