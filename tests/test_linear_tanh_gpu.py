"""tanh of the linear layers and hash heads: as exact as the library's that the embedder's own last layer uses."""
import pytest
import torch

from pixelbox_amd import linear

pytestmark = pytest.mark.gpu

# In units of 2^-24, from |v| = 1 on tanh = 1 - 2 t, t = e / (1 + e), e = exp2(-2 |v| log2 e): e is off by 4 |v| (the constant's and the product's
# rounding) + 2 (exp2), t by that / (1 + e) + 1 (the sum) + 2 (the reciprocal) + 1 (the product); the result takes 2 t / tanh v of it, 0.313 at 1
# and less above (0.313 (6 / 1.135 + 4) = 2.9), and rounds by 1: 3.9.  Below 1 the sum is v + v^3 P: the fit 0.1; v^2, its product with v and P's
# steps at most 5 of the cubic part, which is at most 0.313 of the result; the last step 1: 2.7.
UNITS = 4


def tanh(v):
    return linear.linear_grouped(v[:, None].cuda(), torch.ones((1, 1, 1), device="cuda"), torch.tensor([0, v.numel()], dtype=torch.int32, device="cuda"), act="tanh")[:, 0]


def test_tanh_within_four_units():
    v = torch.cat([torch.linspace(0.2, 1.3, 2_000_000, dtype=torch.float64), torch.linspace(1e-3, 12.0, 1_000_000, dtype=torch.float64),
                   torch.logspace(-30, 2, 200_000, dtype=torch.float64)]).float()
    one = torch.tensor([1.0])
    v = torch.cat([v, torch.nextafter(one, torch.tensor([0.0])), one, torch.nextafter(one, torch.tensor([2.0]))])
    for x in (v, -v):
        want = torch.tanh(x.double())
        units = ((tanh(x).cpu().double() - want) / want).abs() * 2.0 ** 24
        print("worst", units.max().item(), "at", x[units.argmax()].item(), "mean square", units.square().mean().sqrt().item())
        assert units.max().item() <= UNITS


def test_tanh_is_odd_and_ends_at_one():
    v = torch.tensor([0.0, 2e-38, 1e-30, 1e-20, 8.0, 9.1, 20.0, 88.0, 1e30, float("inf")])
    y, minus = tanh(v).cpu(), tanh(-v).cpu()
    assert torch.equal(y, -minus)  # values: the product of -0 is +0, for a sum that starts at +0 is +0 behind -0
    assert torch.equal(y[:4], v[:4]) and (y[5:] == 1.0).all() and torch.isnan(tanh(torch.tensor([float("nan")]))).all()
