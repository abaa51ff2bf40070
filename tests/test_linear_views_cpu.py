"""Operands whose values are not just what lies in their memory: tangents of forward-mode differentiation and negated views are refused."""
import pytest
import torch
from torch.autograd import forward_ad

from pixelbox_amd import linear
from test_linear_cpu import _grouped_args, _i8_args, fake


def dual(t):
    return fake(forward_ad.make_dual(t, torch.ones_like(t)))


def negated(*shape):
    v = torch.ones(shape, dtype=torch.complex64).conj().imag
    assert v.is_neg()
    return fake(v)


@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused_not_lost(grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for name in ("x_scale", "w_scale", "bias", "out"):
            t = dual(torch.zeros((3, 5)) if name == "out" else torch.ones(3 if name == "x_scale" else 5))
            with pytest.raises(ValueError, match="tangent"):
                linear.linear_i8(**{**_i8_args(), name: t})
        for name, shape in (("x", (3, 8)), ("w", (2, 5, 8)), ("bias", (2, 5)), ("out", (3, 5))):
            with pytest.raises(ValueError, match="tangent"):
                linear.linear_grouped(**{**_grouped_args(), name: dual(torch.zeros(shape))})
        with pytest.raises(ValueError, match="tangent"):
            linear.quantize_rows(dual(torch.zeros((3, 8))))
        with pytest.raises(ValueError, match="tangent"):
            linear.quantize_rows(fake(torch.zeros((3, 8))), scale=dual(torch.zeros(3)))
        # the values alone are taken: what is left to refuse them is a missing GPU, or nothing
        plain = forward_ad.unpack_dual(forward_ad.make_dual(torch.zeros((3, 8)), torch.ones((3, 8)))).primal
        linear._no_grad(plain, torch.zeros(3, dtype=torch.int8), None)


def test_a_negated_view_is_refused_not_read_unnegated():
    with pytest.raises(ValueError, match="x is a negated view"):
        linear.quantize_rows(negated(3, 1))
    with pytest.raises(ValueError, match="x is a negated view"):
        linear.linear_grouped(**{**_grouped_args(), "x": negated(3, 1), "w": fake(torch.zeros((2, 5, 1)))})
    with pytest.raises(ValueError, match="w is a negated view"):
        linear.linear_grouped(**{**_grouped_args(), "x": fake(torch.zeros((3, 1))), "w": negated(2, 5, 1)})
    with pytest.raises(ValueError, match="out is a negated view"):
        linear.linear_grouped(**{**_grouped_args(), "w": fake(torch.zeros((2, 1, 8))), "out": negated(3, 1)})
    one = dict(x=fake(torch.zeros((1, 8), dtype=torch.int8)), w=fake(torch.zeros((1, 8), dtype=torch.int8)), w_scale=fake(torch.ones(1)),
               x_scale=fake(torch.ones(1)), out=fake(torch.zeros((1, 1))))
    for name in ("x_scale", "w_scale", "bias"):
        with pytest.raises(ValueError, match=f"{name} is a negated view"):
            linear.linear_i8(**{**one, name: negated(1)})
