"""8-bit products of rows whose scales lie at the ends of f32: finite where the result is, and as exact as elsewhere."""
import pytest
import torch

import linear_ref as ref
from pixelbox_amd import linear

pytestmark = pytest.mark.gpu


def case(m, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    x, w = (torch.randint(-128, 128, s, generator=g, dtype=torch.int32).to(torch.int8).cuda() for s in ((m, k), (n, k)))
    # rows of values from the smallest to the largest float, in turn
    xs = torch.tensor([2.0 ** -149, 3e-41, 2.0 ** -126, 2.0 ** -100, 1e-30, 1.0, 1e28, 2.0 ** 96, 1e33, 2.6e36, 3e38])[torch.arange(m) % 11]
    xs = xs * (1 + torch.rand(m, generator=g) * 0.1)
    # ... and channels that bring most of them back to the middle: results from 2^-149 to beyond the largest float
    ws = torch.tensor([1e-38, 1e-33, 1e-30, 1e-6, 1.0, 1e6, 1e30, 1e36])[torch.arange(n) % 8] * (1 + torch.rand(n, generator=g) * 0.1)
    return x, xs.clamp(max=3.4e38).cuda(), w, ws.cuda()


def check(y, x, xs, w, ws):
    want, bound = ref.linear(x, w, None, "none", torch.float32, xs, ws)
    most = torch.finfo(torch.float32).max
    # beyond the largest float by more than the bound: infinity; within it: either
    y = y.cpu().double()
    far, near = want.abs() - bound > most, want.abs() + bound <= most
    # a result below the smallest normal value may be rounded twice there: half of the smallest value more
    bound = bound + 2.0 ** -150
    assert near.float().mean() > 0.4 and far.any()
    assert (torch.isinf(y) & (torch.sign(y) == torch.sign(want)))[far].all()
    off = (y - want).abs()[near] - bound[near]
    assert not torch.isnan(y).any() and off.max().item() <= 0, (off.max().item(), want[near][off.argmax()].item(), y[near][off.argmax()].item())


# one per kind of kernel: few rows, tiles of 64, 128 and 256
@pytest.mark.parametrize("m,n,k", [(33, 24, 1280), (600, 700, 300), (2500, 2100, 130), (2048, 2048, 2048), (4100, 4096, 96)])
def test_products_at_the_ends_of_the_range(m, n, k):
    x, xs, w, ws = case(m, n, k, m)
    check(linear.linear_i8(x, xs, w, ws), x, xs, w, ws)


def test_a_row_of_large_values_through_codes():
    """values around 10^36, weights around 10^-3: a result far inside the range, whose sum times the row's scale is not"""
    g = torch.Generator().manual_seed(5)
    xf, wf = torch.rand((3, 1280), generator=g) * 1e36, torch.rand((256, 1280), generator=g) * 1e-3
    (x, xs), (w, ws) = linear.quantize_rows(xf.cuda()), linear.quantize_rows(wf.cuda())
    y = linear.linear_i8(x, xs, w, ws)
    assert torch.isfinite(y).all()
    ref.check(y, *ref.linear(x, w, None, "none", torch.float32, xs, ws))
    assert ((y.cpu().double() - xf.double() @ wf.double().t()).abs() <= 0.02 * (xf.double() @ wf.double().t())).all()


def test_scales_that_are_no_number_show():
    x, w = torch.ones((4, 64), dtype=torch.int8, device="cuda"), torch.ones((8, 64), dtype=torch.int8, device="cuda")
    xs = torch.tensor([float("nan"), float("inf"), 0.0, 1.0], device="cuda")
    y = linear.linear_i8(x, xs, w, torch.ones(8, device="cuda")).cpu()
    assert torch.isnan(y[0]).all() and torch.isinf(y[1]).all() and (y[2] == 0).all() and (y[3] == 64).all()
