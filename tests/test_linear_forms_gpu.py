"""Ragged grouped products through every tile kernel (tests/linear_forms.py): row lists that gather and scatter, empty groups, groups of one row, rows
without a group, row numbers that are none -- each row against 64 bits, within the bounds of tests/linear_ref.py."""
import pytest
import torch

import linear_forms as forms
import linear_ref as ref
from pixelbox_amd import capi, linear

pytestmark = pytest.mark.gpu

FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = ref.U


def strided(t, ld):
    """the same rows at a stride of ld elements, with NaN (or 77) between them; starts on 16 bytes"""
    rows, k = t.shape
    buf = torch.full((rows * ld + 16,), 77 if t.dtype == torch.int8 else float("nan"), dtype=t.dtype, device="cuda")
    v = buf.as_strided((rows, k), (ld, 1), 0)
    v.copy_(t)
    return v


def want_and_bound(x, xs, w, ws, b, name, dtype):
    """linear_ref's result and bound, in 64 bits on the GPU"""
    p, size = x.double() @ w.double().t(), None
    if xs is not None:
        p = p * xs.double()[:, None] * ws.double()
        err = 3 * U * p.abs()
    else:
        size = x.double().abs() @ w.double().abs().t()
        err = 2 * x.shape[1] * U * size
    v = p if b is None else p + b.double()
    err = err + U * v.abs()
    y = ref.act(v, name)
    if name == "silu":
        err = 1.1 * err + (3 * v.abs() + 8) * U * y.abs()
    info = torch.finfo(dtype)
    return y, err * 1.01 + (y.abs() + err) * (info.eps / 2) + info.smallest_normal * info.eps / 2


@pytest.mark.parametrize("kind,align,m,groups,n,k,form", forms.CASES)
def test_ragged_groups_through_every_form(kind, align, m, groups, n, k, form):
    assert capi.linear_form(forms.TYPE[kind], m, n, k, groups, align) == form
    g = torch.Generator(device="cuda").manual_seed(m * 31 + n)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    x_total, y_total, ld = m + 9, m + 4, forms.row_stride(kind, k, align)
    xs = ws = None
    if kind == "i8":
        x = torch.randint(-128, 128, (x_total, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
        w = torch.randint(-128, 128, (groups * n, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
        xs = torch.rand((x_total,), generator=g, device="cuda") * 0.02 + 1e-3
        ws = torch.rand((groups, n), generator=g, device="cuda") * 0.02 / k ** 0.5
    else:
        x, w = normal(x_total, k).to(FLOATS[kind]), (normal(groups * n, k) * k ** -0.5).to(FLOATS[kind])
    b = normal(groups, n)
    x, w = strided(x, ld), strided(w, ld)
    w3 = w.as_strided((groups, n, k), (n * ld, ld, 1), 0)
    # groups of very different sizes; group 1 has no row, the last one has one, one row in twenty has no group
    share = torch.rand(groups, generator=g, device="cuda") ** 2 + 0.02
    share[1], share[-1] = 0.0, 0.0
    group = torch.multinomial(share, m, replacement=True, generator=g).to(torch.int32)
    group[torch.rand(m, generator=g, device="cuda") < 0.05] = -1
    group[m // 2] = groups - 1
    offsets, order = linear.group_rows(group, groups)
    # rows of x in any order, some twice, some none; rows of y in another order, each once, some none
    x_rows = torch.randperm(x_total, generator=g, device="cuda")[:m].to(torch.int32)
    x_rows[5::53] = x_rows[4::53][: x_rows[5::53].numel()]
    x_rows[7::41], x_rows[9::97] = -1, x_total
    y_rows = torch.randperm(y_total, generator=g, device="cuda")[:m].to(torch.int32)
    y_rows[3::61], y_rows[8::67] = -3, y_total
    cuts = offsets.tolist()
    assert cuts[1] == cuts[2] and cuts[-1] - cuts[-2] == 1 and cuts[-1] < m
    live = (x_rows >= 0) & (x_rows < x_total) & (y_rows >= 0) & (y_rows < y_total)
    for name, dtype, bias in (("none", FLOATS.get(kind, torch.float16), None), ("silu", torch.float32, b)):
        out = torch.full((y_total + 2, n), 3.0, dtype=dtype, device="cuda")
        linear.linear_grouped(x, w3, offsets, x_rows=x_rows, y_rows=y_rows, x_scale=xs, w_scale=ws, bias=bias, act=name, out=out[1:-1])
        left = torch.ones(y_total + 2, dtype=torch.bool, device="cuda")
        for gi in range(groups):
            at = torch.arange(cuts[gi], cuts[gi + 1], device="cuda")
            at = at[live[at]]
            if at.numel() == 0:
                continue
            xr, yr = x_rows[at].long(), y_rows[at].long() + 1
            want, bound = want_and_bound(x[xr], None if xs is None else xs[xr], w3[gi], None if ws is None else ws[gi], None if bias is None else bias[gi], name, dtype)
            off = (out[yr].double() - want).abs() - bound
            assert not torch.isnan(off).any() and off.max().item() <= 0, (name, gi, off.max().item(), off.argmax().item())
            left[yr] = False
        assert (out[left] == 3.0).all() and left.sum() > m // 20, name
        # the order of the groups, as a batch of heads or experts has it: rows of x read and of y written by the same list
        if name == "silu":
            same = torch.full((m, n), 3.0, device="cuda")
            linear.linear_grouped(x[:m], w3, offsets, rows=order, x_scale=None if xs is None else xs[:m], w_scale=ws, bias=b, act=name, out=same)
            for gi in {0, groups // 2, groups - 1}:
                r = (group == gi).nonzero().squeeze(1)
                want, bound = want_and_bound(x[r], None if xs is None else xs[r], w3[gi], None if ws is None else ws[gi], b[gi], name, torch.float32)
                assert ((same[r].double() - want).abs() <= bound).all(), gi
            assert (same[group < 0] == 3.0).all()
