"""The compiled short way leaves operands with tangents and negated views alone, and they are refused behind it."""
import pytest
import torch
from torch.autograd import forward_ad

from pixelbox_amd import linear

pytestmark = pytest.mark.gpu


def i8(m=6, n=8, k=32):
    x, w = (torch.ones(s, dtype=torch.int8, device="cuda") for s in ((m, k), (n, k)))
    return [x, torch.ones(m, device="cuda"), w, torch.ones(n, device="cuda"), torch.ones(n, device="cuda"), 0, torch.zeros((m, n), device="cuda")]


def test_tangents():
    short = linear._load()
    assert short
    ok = i8()
    x, w = torch.ones((6, 32), device="cuda"), torch.ones((1, 8, 32), device="cuda")
    offsets = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    codes, scale = torch.empty((6, 32), dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda")
    grouped = [x, w, offsets, None, None, None, None, torch.ones((1, 8), device="cuda"), 0, torch.zeros((6, 8), device="cuda")]
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        assert short.linear_i8(*ok) == 0 and short.linear_grouped(*grouped) == 0 and short.quantize_rows(x, codes, scale) == 0
        for i in (1, 3, 4, 6):
            assert short.linear_i8(*ok[:i], dual(ok[i]), *ok[i + 1:]) is None, i
        for i in (0, 1, 7, 9):
            assert short.linear_grouped(*grouped[:i], dual(grouped[i]), *grouped[i + 1:]) is None, i
        assert short.quantize_rows(dual(x), codes, scale) is None and short.quantize_rows(x, codes, dual(scale)) is None
        with pytest.raises(ValueError, match="tangent"):
            linear.linear_grouped(dual(x), w, offsets, out=grouped[9])
        with pytest.raises(ValueError, match="tangent"):
            linear.linear_i8(*ok[:4], out=dual(ok[6]))
        with pytest.raises(ValueError, match="tangent"):
            linear.quantize_rows(dual(x), codes=codes, scale=scale)
        # the values alone
        y = linear.linear_grouped(forward_ad.unpack_dual(dual(x)).primal, w, offsets)
        assert (y == 32).all()


def test_negated_views():
    short = linear._load()
    ok = i8(1, 1)
    minus = torch.ones(1, dtype=torch.complex64, device="cuda").conj().imag
    assert minus.is_neg() and minus.is_contiguous()
    assert short.linear_i8(*ok) == 0
    for i in (1, 3, 4):
        assert short.linear_i8(*ok[:i], minus, *ok[i + 1:]) is None, i
    with pytest.raises(ValueError, match="x_scale is a negated view"):
        linear.linear_i8(ok[0], minus, *ok[2:4], out=ok[6])
    column = torch.ones((6, 1), dtype=torch.complex64, device="cuda").conj().imag
    with pytest.raises(ValueError, match="x is a negated view"):
        linear.quantize_rows(column)
    c, s = linear.quantize_rows(column.resolve_neg())
    assert (c == 0).all()  # the imaginary part of 1
