"""The linear layers on device buffers against 64-bit references (tests/linear_ref.py): every type, odd sizes, strides, alignments, ragged and
empty groups, rows that no group has, streams, graphs and threads."""
import threading

import pytest
import torch

import linear_ref as ref
from pixelbox_amd import capi, linear

pytestmark = pytest.mark.gpu

FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
KINDS = ["f32", "bf16", "f16", "i8"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def codes(shape, g):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int32).to(torch.int8).cuda()


def strided(t, ld, shift=0):
    """the same rows at a stride of ld elements, starting `shift` elements into a buffer that holds NaN (or 77) everywhere else"""
    m, k = t.shape
    fill = 77 if t.dtype == torch.int8 else float("nan")
    buf = torch.full((shift + max(m, 1) * ld + 64,), fill, dtype=t.dtype, device=t.device)
    v = buf.as_strided((m, k), (ld, 1), shift)
    v.copy_(t)
    return v


# ---- quantize_rows -----------------------------------------------------------------------------------------------------------------------

def check_codes(x, c, s):
    want_c, want_s = ref.quantize(x)
    assert torch.equal(s.cpu().view(torch.int32)[~torch.isnan(want_s)], want_s.view(torch.int32)[~torch.isnan(want_s)])
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(want_s))
    assert torch.equal(c.cpu(), want_c)


@pytest.mark.parametrize("kind", list(FLOATS))
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (2, 64), (5, 255), (4, 1280), (3, 1289), (2, 4096), (2, 8192), (2, 8200), (1, 20011), (700, 33)])
def test_quantize_rows_is_exact(kind, m, k):
    x = rand((m, k), FLOATS[kind], gen(m * 10007 + k), 3.0)
    check_codes(x, *linear.quantize_rows(x))


@pytest.mark.parametrize("kind", list(FLOATS))
def test_quantize_rows_strides_and_alignment(kind):
    x = rand((9, 301), FLOATS[kind], gen(5))
    for ld, shift in ((301, 1), (304, 0), (320, 3), (512, 8)):
        v = strided(x, ld, shift)
        c = strided(torch.zeros((9, 301), dtype=torch.int8, device="cuda"), ld + 7, shift)
        c2, s = linear.quantize_rows(v, codes=c)
        assert c2 is c
        check_codes(x, c, s)
        flat = c.as_strided((9 * (ld + 7),), (1,), shift).view(9, ld + 7)
        assert (flat[:-1, 301:] == 77).all()  # what lies between the rows is left alone


def test_quantize_rows_special_rows():
    x = torch.zeros((10, 300))
    x[1, 5] = float("inf")
    x[2, 299] = float("nan")
    x[3] = 2.0 ** -149            # every value subnormal
    x[4, 0] = 3.4e38
    x[5] = torch.arange(300) - 150.0
    x[6] = 127.0                  # scale 1
    x[6, 1:] = torch.arange(299) % 100 + 0.5   # halves to even
    x[7] = -x[6]
    x[8] = 2.0 ** -126
    x[9, 17] = -float("inf")
    c, s = linear.quantize_rows(x.cuda())
    check_codes(x, c, s)
    assert (c[0] == 0).all() and (c[[1, 2, 9]] == 0).all() and torch.isnan(s[[1, 2, 9]]).all()
    assert c[6, 1:7].tolist() == [0, 2, 2, 4, 4, 6]


def test_quantize_rows_next_to_halves():
    # values whose quotient is within a unit of f32 of a half: what a rounded quotient decides by luck
    g = gen(11)
    rows = []
    for _ in range(64):
        top = (torch.rand(1, generator=g) * 10 + 0.1).float()
        s = (top.double() / 127).float()
        r = torch.randint(0, 126, (400,), generator=g).double() + 0.5
        v = (r * s.double()).float()
        v = torch.nextafter(v, torch.where(torch.rand(400, generator=g) < 0.5, torch.tensor(0.0), torch.tensor(1e9)))
        rows.append(torch.cat([top, v.clamp(max=float(top)), (r * s.double()).float().clamp(max=float(top))]))
    x = torch.stack(rows)
    check_codes(x, *linear.quantize_rows(x.cuda()))


def test_quantize_rows_nothing():
    c, s = linear.quantize_rows(torch.empty((0, 5), device="cuda"))
    assert c.shape == (0, 5) and s.shape == (0,)
    c, s = linear.quantize_rows(torch.empty((3, 0), device="cuda"))
    assert c.shape == (3, 0) and (s == 2.0 ** -126).all()


# ---- linear_i8 ---------------------------------------------------------------------------------------------------------------------------

def i8_case(m, n, k, seed, bias=True):
    g = gen(seed)
    x, w = codes((m, k), g), codes((n, k), g)
    xs, ws = (torch.rand((m,), generator=g) * 0.02 + 1e-3).cuda(), (torch.rand((n,), generator=g) * 0.02 / max(k, 1) ** 0.5).cuda()
    return x, xs, w, ws, rand((n,), torch.float32, g) if bias else None


SIZES = [(1, 1, 1), (1, 256, 1280), (2, 17, 15), (3, 16, 16), (16, 64, 63), (17, 33, 64), (5, 1000, 129), (31, 48, 300), (64, 64, 128), (65, 130, 257),
         (100, 1000, 1289), (257, 129, 1000), (1000, 700, 384), (4, 2048, 5000), (130, 4096, 640), (2049, 1025, 96)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_i8(m, n, k):
    x, xs, w, ws, b = i8_case(m, n, k, m + n + k)
    for name, dt, bias in (("none", torch.float32, None), ("silu", torch.float16, b), ("tanh", torch.bfloat16, b)):
        y = linear.linear_i8(x, xs, w, ws, bias=bias, act=name, dtype=dt)
        assert y.dtype == dt
        ref.check(y, *ref.linear(x, w, bias, name, dt, xs, ws), (m, n, k, name))


# sizes that each form of the product is chosen for (16 x 16, 32 x 16 and 32 x 32 outputs per workgroup with K split over its waves; tiles of 64,
# 128 with four and with two LDS stages, 256), K around whole steps of 128 bytes and around the stages' number, rows on 16 bytes and not
FORM_SIZES = [(16, 4096), (32, 4096), (60, 4000), (300, 1000), (1000, 4000), (2048, 4090), (4000, 4096)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n", FORM_SIZES)
def test_every_form_at_every_remainder(kind, m, n):
    size = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}[kind]
    most = 1040 // size
    x, xs, w, ws, b = grouped_case(kind, m, 1, n, most, m + n)
    offsets = torch.tensor([0, m], dtype=torch.int32).cuda()
    rows = gen(3)
    pick = torch.randperm(m, generator=rows)[:70]  # rows that are compared with 64 bits; all are compared with one another's K below
    for k in [most, 512 // size, 512 // size + 1, 640 // size - 1, 128 // size, 128 // size + 3, 256 // size, 5]:
        xk, wk = x[:, :k], w[:, :, :k]
        if k == most - 0:
            xk, wk = x, w
        if k % 2:
            xk, wk = xk.contiguous(), wk.contiguous()
        y = torch.full((m, n), float("nan"), device="cuda")
        linear.linear_grouped(xk, wk, offsets, x_scale=xs, w_scale=ws, bias=b, out=y)
        assert not torch.isnan(y).any(), k
        ref.check(y[pick.cuda()], *ref.linear(x.cpu()[pick][:, :k], w[0, :, :k], b[0], "none", torch.float32, None if xs is None else xs.cpu()[pick],
                                              None if ws is None else ws[0]), (m, n, k))
        # every row and channel against the same product on the GPU in 64 bits: order of sums aside, the same
        want = x[:, :k].double() @ w[0, :, :k].double().t()
        if kind == "i8":
            want = want * xs.double()[:, None] * ws[0].double()
        want += b[0].double()
        scale = want.abs().amax().item()
        assert (y.double() - want).abs().amax().item() <= 2e-5 * scale


# the forms that the sizes above leave out for some type or alignment
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n", [(24, 3000), (300, 2048), (1300, 1400), (1000, 4096), (2048, 2048), (1500, 3000), (3000, 3001)])
def test_every_form_at_every_alignment(kind, m, n):
    size = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}[kind]
    k = 1040 // size
    x, xs, w, ws, b = grouped_case(kind, m, 1, n, k, m + n)
    want = x.double() @ w[0].double().t()
    if kind == "i8":
        want = want * xs.double()[:, None] * ws[0].double()
    want += b[0].double()
    # a sum of k products rounds at most k times, each time by a unit (2 x 2^-24) of at most the sum of the products' magnitudes; scales,
    # bias and the 64-bit result's own products: less than 8 x 2^-24 more
    most = (2 * k + 8) * 2.0 ** -24 * (x.double().abs() @ w[0].double().abs().t() * (1 if xs is None else xs.double()[:, None] * ws[0].double()) + b[0].double().abs())
    offsets = torch.tensor([0, m], dtype=torch.int32).cuda()
    for ld, shift in ((k, 0), (k + 16 // size, 16 // size), (k + 4 // size, 0), (k, 4 // size), (k + 1, 0), (k + 8 // size, 1)):
        y = torch.full((m, n), float("nan"), device="cuda")
        wl = strided(w[0], ld, shift)
        linear.linear_grouped(strided(x, ld, shift), wl.as_strided((1, n, k), (n * ld, ld, 1), wl.storage_offset()), offsets, x_scale=xs, w_scale=ws, bias=b, out=y)
        assert ((y.double() - want).abs() <= most).all(), (ld, shift)


def test_linear_i8_sums_are_exact_at_the_largest_k():
    k = capi.PB_LINEAR_I8_MAX_K
    x = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    x[1] = 127
    w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    w[2] = 127
    one2, one3 = torch.ones(2, device="cuda"), torch.ones(3, device="cuda")
    y = linear.linear_i8(x, one2, w, one3)
    want = (x.cpu().double() @ w.cpu().double().T).float()
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_i8_strides_and_alignment(m):
    n, k = 203, 301
    x, xs, w, ws, b = i8_case(m, n, k, 3)
    want = ref.linear(x, w, b, "none", torch.float16, xs, ws)
    base = linear.linear_i8(x, xs, w, ws, bias=b, dtype=torch.float16)
    for ld, shift in ((301, 1), (304, 0), (304, 16), (320, 5), (336, 16)):
        out = strided(torch.zeros((m, n), dtype=torch.float16, device="cuda"), n + 5, shift)
        y = linear.linear_i8(strided(x, ld, shift), xs, strided(w, ld, shift), ws, bias=b, out=out)
        assert y is out
        ref.check(y, *want)
        assert torch.equal(y, base)  # exact sums: the same bits by every way
        assert torch.isnan(out.as_strided((m - 1, 5), (n + 5, 1), shift + n)).all()


def test_linear_i8_rows_do_not_depend_on_the_batch():
    x, xs, w, ws, b = i8_case(1500, 640, 1280, 9)
    y = linear.linear_i8(x, xs, w, ws, bias=b, act="tanh")
    for i in (0, 1, 777, 1499):
        assert torch.equal(linear.linear_i8(x[i:i + 1], xs[i:i + 1], w, ws, bias=b, act="tanh")[0], y[i])
    assert torch.equal(linear.linear_i8(x[100:190], xs[100:190], w, ws, bias=b, act="tanh"), y[100:190])


def test_linear_i8_nothing():
    x, xs, w, ws, b = i8_case(4, 6, 32, 1)
    assert linear.linear_i8(x[:0], xs[:0], w, ws).shape == (0, 6)
    assert linear.linear_i8(x, xs, w[:0], ws[:0]).shape == (4, 0)
    y = linear.linear_i8(x[:, :0], xs, w[:, :0], ws, bias=b)
    assert torch.equal(y, b.expand(4, 6))


def test_a_row_with_a_nan_stays_alone():
    g = gen(2)
    x = rand((70, 500), torch.float32, g)
    x[3, 7], x[50, 499] = float("nan"), float("inf")
    w, ws = linear.quantize_rows(rand((90, 500), torch.float32, g))
    y = linear.linear_i8(*linear.quantize_rows(x), w, ws)
    assert torch.isnan(y[[3, 50]]).all() and torch.isfinite(y[[i for i in range(70) if i not in (3, 50)]]).all()


def test_linear_i8_rows_beyond_32_bits():
    k, n, m, ld = 300, 40, 3, (1 << 31) + 48
    x, xs, w, ws, b = i8_case(m, n, k, 21)
    buf = torch.empty((m - 1) * ld + k, dtype=torch.int8, device="cuda")
    far = buf.as_strided((m, k), (ld, 1))
    far.copy_(x)
    out = torch.empty((m - 1) * ld + n, dtype=torch.float16, device="cuda").as_strided((m, n), (ld, 1))
    linear.linear_i8(far, xs, w, ws, bias=b, out=out)
    ref.check(out, *ref.linear(x, w, b, "none", torch.float16, xs, ws))
    c, s = linear.quantize_rows(out, codes=far[:, :n])
    check_codes(out, c, s)


def test_more_rows_than_one_launch_has_threads_for():
    """quantize_rows: in several launches; linear_i8: by larger tiles.  Few values and channels, rows by the hundred million"""
    m, k = 40_000_000, 2
    x = torch.empty((m, k), dtype=torch.float16, device="cuda")
    r = torch.arange(m, device="cuda")
    x[:, 0] = (r % 1009 + 1).to(torch.float16)
    x[:, 1] = -(r % 127).to(torch.float16)
    c, s = linear.quantize_rows(x)
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, m - 5, m - 1], device="cuda")
    check_codes(x[at], c[at], s[at])
    by = torch.full((1,), 127.0, device="cuda")  # a tensor: torch divides by a number by multiplying with its reciprocal
    assert torch.equal(s, torch.clamp(torch.maximum(x[:, 0], -x[:, 1]).float() / by, min=2.0 ** -126))
    del x, c, s, r
    m = 140_000_000  # 16 rows a workgroup of 512 threads would be more than 2^32 threads
    x = (torch.arange(m, device="cuda") % 251 - 125).to(torch.int8)[:, None]
    one = torch.ones(m, device="cuda")
    w, ws = torch.tensor([[3]], dtype=torch.int8, device="cuda"), torch.tensor([0.5], device="cuda")
    y = linear.linear_i8(x, one, w, ws, dtype=torch.float16)
    assert torch.equal(y, x.to(torch.float16) * 1.5)  # 375 / 2 at most: halves, exact in f16


# ---- group_rows --------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,groups", [(0, 3), (1, 1), (1, 5), (63, 2), (64, 64), (257, 7), (4096, 1024), (5000, 33), (20001, 300)])
@pytest.mark.parametrize("shift", [0, 1])
def test_group_rows(m, groups, shift):
    g = torch.randint(-2, groups + 3, (m + shift,), generator=gen(m + groups), dtype=torch.int32).cuda()[shift:]
    offsets, order = linear.group_rows(g, groups)
    want_offsets, want_order = ref.group(g, groups)
    assert torch.equal(offsets.cpu(), want_offsets) and torch.equal(order.cpu(), want_order)


@pytest.mark.parametrize("m", [131072, 131073, 400000])
def test_group_rows_of_more_than_one_chunk(m):
    groups = 5
    g = torch.randint(-1, groups + 1, (m,), generator=gen(m), dtype=torch.int32).cuda()
    offsets, order = linear.group_rows(g, groups)
    key = torch.where((g >= 0) & (g < groups), g, torch.full_like(g, groups)).cpu()
    assert torch.equal(order.cpu().long(), torch.argsort(key, stable=True))
    assert offsets.cpu().tolist() == [int((key < i).sum()) for i in range(groups + 1)]


@pytest.mark.parametrize("value", [-1, 0, 2, 3, 2**31 - 1, -2**31])
def test_group_rows_all_alike(value):
    g = torch.full((777,), value, dtype=torch.int32, device="cuda")
    offsets, order = linear.group_rows(g, 3)
    assert torch.equal(order.cpu(), torch.arange(777, dtype=torch.int32))
    assert offsets.cpu().tolist() == [0] + [777 if 0 <= value <= i else 0 for i in range(3)]


@pytest.mark.parametrize("m", [100, 3001, 20000, 32769, 60000, 65537, 100001, 131072, 150000])
@pytest.mark.parametrize("groups", [1, 2, 4, 6])
def test_group_rows_of_dense_and_sparse_groups(m, groups):
    """one group with most rows, in runs and single, beside small ones: both ways of writing a group's rows"""
    g = torch.randint(0, 40, (m,), generator=gen(m + groups), dtype=torch.int32)
    g = torch.where(g < groups, g, torch.zeros_like(g))
    g[m // 3: m // 2] = groups - 1
    g[m // 2: m // 2 + m // 7] = -1
    offsets, order = linear.group_rows(g.cuda(), groups)
    want_offsets, want_order = ref.group(g, groups)
    assert torch.equal(offsets.cpu(), want_offsets) and torch.equal(order.cpu(), want_order)


# ---- linear_grouped ----------------------------------------------------------------------------------------------------------------------

def grouped_case(kind, m, groups, n, k, seed, bias=True):
    g = gen(seed)
    if kind == "i8":
        x, w = codes((m, k), g), codes((groups, n, k), g)
        xs = (torch.rand((m,), generator=g) * 0.02 + 1e-3).cuda()
        ws = (torch.rand((groups, n), generator=g) * 0.02 / max(k, 1) ** 0.5).cuda()
    else:
        x, w, xs, ws = rand((m, k), FLOATS[kind], g), rand((groups, n, k), FLOATS[kind], g, max(k, 1) ** -0.5), None, None
    return x, xs, w, ws, rand((groups, n), torch.float32, g) if bias else None


def some_groups(m, groups, seed, none=0.1, skew=True):
    g = gen(seed)
    p = torch.rand(groups, generator=g) ** (6 if skew else 1) + 1e-9
    v = torch.multinomial(p, max(m, 1), replacement=True, generator=g)[:m].to(torch.int32)
    v[torch.rand(m, generator=g) < none] = -1
    return v.cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,groups,n,k", [(1, 1, 1, 1), (1, 9, 33, 100), (7, 3, 16, 31), (40, 64, 130, 64), (300, 5, 257, 129), (513, 8, 256, 320),
                                          (1000, 3, 100, 1001), (3000, 2, 640, 96), (2500, 70, 65, 72)])
def test_linear_grouped(kind, m, groups, n, k):
    x, xs, w, ws, b = grouped_case(kind, m, groups, n, k, m + k)
    offsets, order = linear.group_rows(some_groups(m, groups, n), groups)
    for name, dt, bias in (("none", torch.float32, None), ("tanh" if m % 2 else "silu", torch.bfloat16 if k % 2 else torch.float16, b)):
        out = torch.full((m, n), 3.0, dtype=dt, device="cuda")
        y = linear.linear_grouped(x, w, offsets, rows=order, x_scale=xs, w_scale=ws, bias=bias, act=name, out=out)
        assert y is out
        ref.check(y, *ref.grouped(x, w, offsets, order, order, bias, name, torch.full((m, n), 3.0, dtype=dt), xs, ws), (kind, m, groups, n, k, name))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [50, 2000])
def test_linear_grouped_without_row_lists(kind, m):
    groups, n, k = 6, 70, 200
    x, xs, w, ws, b = grouped_case(kind, m, groups, n, k, 4)
    cuts = torch.tensor([0, 0, m // 7, m // 7, m // 2, m - 3, m - 3], dtype=torch.int32).cuda()  # three empty groups, three rows of no group
    out = torch.full((m + 2, n), -5.0, device="cuda")
    linear.linear_grouped(x, w, cuts, x_scale=xs, w_scale=ws, bias=b, out=out)
    ref.check(out, *ref.grouped(x, w, cuts, None, None, b, "none", torch.full((m + 2, n), -5.0), xs, ws))
    assert (out[m - 3:] == -5.0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_linear_grouped_strides_and_alignment(kind):
    m, groups, n, k = 333, 4, 51, 77
    x, xs, w, ws, b = grouped_case(kind, m, groups, n, k, 14)
    offsets, order = linear.group_rows(some_groups(m, groups, 2), groups)
    for ld, shift in ((77, 1), (80, 0), (96, 16), (81, 3)):
        wv = strided(w.view(groups * n, k), ld, shift).as_strided((groups, n, k), (n * ld, ld, 1), shift)
        out = strided(torch.zeros((m, n), dtype=torch.bfloat16, device="cuda"), n + 3, shift)
        linear.linear_grouped(strided(x, ld, shift), wv, offsets, rows=order, x_scale=xs, w_scale=ws, bias=b, act="silu", out=out)
        ref.check(out, *ref.grouped(x, w, offsets, order, order, b, "silu", torch.zeros((m, n), dtype=torch.bfloat16), xs, ws), (ld, shift))


@pytest.mark.parametrize("kind", KINDS)
def test_bad_device_data_touches_nothing_else(kind):
    # offsets outside the rows, groups that run backwards, row numbers outside x and y: skipped, never read or written
    m, groups, n, k = 200, 4, 40, 64
    x, xs, w, ws, _ = grouped_case(kind, m, groups, n, k, 8)
    offsets = torch.tensor([-50, 60, 30, 2**31 - 1, 5], dtype=torch.int32).cuda()
    rows = torch.arange(m, dtype=torch.int32).cuda()
    rows[::7], rows[1::7] = -1, 2**31 - 1
    rows[3::7] = m
    out = torch.full((m, n), 9.0, device="cuda")
    linear.linear_grouped(x, w, offsets, rows=rows, x_scale=xs, w_scale=ws, out=out)
    o = torch.tensor([0, 60, 30, m, 5])
    want, bound = torch.full((m, n), 9.0, dtype=torch.float64), torch.zeros((m, n), dtype=torch.float64)
    for g in range(groups):
        for r in range(int(o[g]), int(o[g + 1])):
            if 0 <= int(rows[r]) < m:
                i = int(rows[r])
                want[i:i + 1], bound[i:i + 1] = ref.linear(x[i:i + 1], w[g], None, "none", torch.float32, None if xs is None else xs[i:i + 1],
                                                           None if ws is None else ws[g])
    ok = (out.cpu().double() - want).abs() <= bound
    # rows 30 .. 59 are listed by groups 0 and 2: either result stands
    twice = [int(rows[r]) for r in range(30, 60) if 0 <= int(rows[r]) < m]
    ok[twice] = True
    assert ok.all()


@pytest.mark.parametrize("name", ["tanh", "silu"])
def test_activations_over_their_range(name):
    """one value, one channel of weight 1: the activation of exactly that value; around 0.4, where tanh changes its formula, closely"""
    v = torch.cat([torch.logspace(-30, 2, 150_000, dtype=torch.float64), torch.linspace(0.3999, 0.4001, 20_000, dtype=torch.float64),
                   torch.linspace(0.01, 12.0, 100_000, dtype=torch.float64)]).float()
    v = torch.cat([v, -v])
    y = linear.linear_grouped(v[:, None].cuda(), torch.ones((1, 1, 1), device="cuda"), torch.tensor([0, v.numel()], dtype=torch.int32, device="cuda"), act=name)
    x = v.double()
    want = ref.act(x, name)
    factor = 9 if name == "tanh" else 3 * x.abs() + 8  # the bounds of linear_ref, and half a unit for a result that no f32 is
    # results below the smallest normal value may be zero; SiLU = v / (1 + e^-v): the reciprocal may be, below 2^-126 (v < -87.3), and
    # times |v| that is all of the result
    below = 2.0 ** -126 * (1 if name == "tanh" else torch.clamp(x.abs(), min=1.0))
    assert ((y[:, 0].cpu().double() - want).abs() <= (factor + 1) * 2.0 ** -24 * want.abs() + below).all()
    ends = torch.tensor([0.0, -0.0, float("inf"), 3e38, -3e38, float("nan")])
    y = linear.linear_grouped(ends[:, None].cuda(), torch.ones((1, 1, 1), device="cuda"), torch.tensor([0, 6], dtype=torch.int32, device="cuda"), act=name)[:, 0].cpu()
    assert y[0] == 0 and y[1] == 0 and torch.isnan(y[5])
    assert y[2:5].tolist() == ([1.0, 1.0, -1.0] if name == "tanh" else [float("inf"), ends[3].item(), 0.0])


def test_rows_of_x_may_be_listed_often():
    x, _, w, _, b = grouped_case("bf16", 5, 3, 64, 128, 6)
    xr = torch.tensor([4, 4, 4, 0, 1, 1, 2, 4], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 3, 5, 8], dtype=torch.int32).cuda()
    y = linear.linear_grouped(x, w, offsets, x_rows=xr, bias=b, dtype=torch.float32)
    assert y.shape == (8, 64)
    ref.check(y, *ref.grouped(x, w, offsets, xr, None, b, "none", torch.zeros((8, 64)), None, None))


def test_a_nan_or_infinity_stays_in_its_row_and_group():
    x, _, w, _, _ = grouped_case("bf16", 100, 2, 48, 100, 16)
    x[10, 3], x[60, 99] = float("nan"), float("inf")
    w[1, 5, 7] = float("nan")
    offsets = torch.tensor([0, 50, 100], dtype=torch.int32).cuda()
    y = linear.linear_grouped(x, w, offsets)
    bad = torch.zeros((100, 48), dtype=torch.bool)
    bad[10], bad[60], bad[50:, 5] = True, True, True
    assert torch.equal(~torch.isfinite(y.cpu()), bad)


# ---- together ----------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
def test_two_layers_of_experts(kind):
    """rows -> their groups -> first layer (gathered, packed) -> [codes ->] second layer (packed, scattered back): each step on what the one
    before it really gave"""
    m, groups, k, h, n = 700, 6, 192, 260, 72
    g = gen(33)
    group = some_groups(m, groups, 7)
    offsets, order = linear.group_rows(group, groups)
    xf = rand((m, k), torch.float32 if kind == "i8" else FLOATS[kind], g)
    w1, w2 = (rand(s, torch.float32, g, s[-1] ** -0.5) for s in ((groups, h, k), (groups, n, h)))
    b1, b2 = rand((groups, h), torch.float32, g), rand((groups, n), torch.float32, g)
    s1 = s2 = xs = hs = None
    if kind == "i8":
        (w1, s1), (w2, s2) = ((c.view(w.shape), s.view(w.shape[:2])) for w in (w1, w2) for c, s in [linear.quantize_rows(w.view(-1, w.shape[-1]))])
        x, xs = linear.quantize_rows(xf)
    else:
        x, w1, w2 = xf, w1.to(xf.dtype), w2.to(xf.dtype)
    mid = linear.linear_grouped(x, w1, offsets, x_rows=order, x_scale=xs, w_scale=s1, bias=b1, act="silu", dtype=torch.float32 if kind == "i8" else None)
    ref.check(mid, *ref.grouped(x, w1, offsets, order, None, b1, "silu", torch.zeros_like(mid).cpu(), xs, s1))
    midq = mid
    if kind == "i8":
        midq, hs = linear.quantize_rows(mid)
        check_codes(mid, midq, hs)
    y = linear.linear_grouped(midq, w2, offsets, y_rows=order, x_scale=hs, w_scale=s2, bias=b2, act="tanh", dtype=torch.float32)
    ref.check(y, *ref.grouped(midq, w2, offsets, None, order, b2, "tanh", torch.zeros_like(y).cpu(), hs, s2))
    assert (y[group == -1] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(kind):
    m, groups, n, k = 400, 5, 96, 160
    x, xs, w, ws, b = grouped_case(kind, m, groups, n, k, 50)
    xf = rand((m, k), torch.float32, gen(51))
    group = some_groups(m, groups, 52)
    offsets, order = linear.group_rows(group, groups)
    out = torch.zeros((m, n), device="cuda")
    c, s = linear.quantize_rows(xf)

    def step():
        linear.group_rows(group, groups, offsets=offsets, order=order)
        if kind == "i8":
            linear.quantize_rows(xf, codes=c, scale=s)
        linear.linear_grouped(c if kind == "i8" else x, w, offsets, rows=order, x_scale=s if kind == "i8" else None, w_scale=ws, bias=b, act="silu", out=out)

    step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for gr in graphs:
        with torch.cuda.graph(gr):
            step()
    for i in range(6):
        xf.copy_(rand((m, k), torch.float32, gen(60 + i)))
        group.copy_(some_groups(m, groups, 70 + i))
        if kind != "i8":
            x.copy_(xf)
        out.zero_()
        step()
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_offsets_that_do_not_ascend_stay_inside():
    """groups that overlap, run backwards or end before they begin: some rows are written more than once or never, none outside"""
    m, groups, n, k = 500, 8, 40, 64
    x, xs, w, ws, b = grouped_case("bf16", m, groups, n, k, 5)
    for bad in ([0, 500, 0, 500, 0, 500, 0, 500, 0], [500, 400, 300, 200, 100, 50, 20, 10, 0], [-(2**31), 2**31 - 1, 7, 9, 9, 2**31 - 1, -1, 3, 500]):
        out = torch.full((m + 20, n), 5.0, device="cuda")
        linear.linear_grouped(x, w, torch.tensor(bad, dtype=torch.int32, device="cuda"), bias=b, out=out[10:m + 10])
        assert (out[:10] == 5).all() and (out[m + 10:] == 5).all() and torch.isfinite(out).all()


def test_another_stream_and_two_threads():
    x, xs, w, ws, b = i8_case(600, 500, 700, 77)
    want = linear.linear_i8(x, xs, w, ws, bias=b, act="tanh")
    torch.cuda.synchronize()
    got, failed = {}, []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                xi = torch.zeros_like(x)
                for _ in range(20):
                    xi.copy_(x)                       # queued on the same stream: the product has to wait for it
                    y = linear.linear_i8(xi, xs, w, ws, bias=b, act="tanh")
                    xi.zero_()
            st.synchronize()
            got[i] = y
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert all(torch.equal(got[i], want) for i in range(2))


def test_no_gradient_is_refused_not_lost():
    x = torch.randn((4, 8), device="cuda", requires_grad=True)
    w = torch.randn((1, 5, 8), device="cuda")
    offsets = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="no gradient"):
        linear.linear_grouped(x, w, offsets)
    with pytest.raises(ValueError, match="no gradient"):
        linear.quantize_rows(x)
    with torch.no_grad():
        assert linear.linear_grouped(x, w, offsets).shape == (4, 5)


@pytest.mark.parametrize("short", [True, False])
def test_a_backward_pass_sees_that_an_output_was_written(short, monkeypatch):
    if not short:
        monkeypatch.setattr(linear, "_compiled", False)
    x, xs, w, ws, b = i8_case(6, 8, 32, 1)
    a, out = torch.ones((6, 8), device="cuda", requires_grad=True), torch.ones((6, 8), device="cuda")
    loss = (a * out).sum()  # saves out
    linear.linear_i8(x, xs, w, ws, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    before = [t._version for t in (out, xs)]
    linear.linear_grouped(x, w[None], torch.tensor([0, 6], dtype=torch.int32, device="cuda"), x_scale=xs, w_scale=ws[None], out=out)
    assert [t._version for t in (out, xs)] == [before[0] + 1, before[1]]
    codes_, scale = linear.quantize_rows(out)
    v = codes_._version, scale._version
    linear.quantize_rows(out, codes=codes_, scale=scale)
    offsets, order = linear.group_rows(torch.zeros(5, dtype=torch.int32, device="cuda"), 1)
    u = offsets._version, order._version
    linear.group_rows(torch.zeros(5, dtype=torch.int32, device="cuda"), 1, offsets=offsets, order=order)
    assert (codes_._version, scale._version) == (v[0] + 1, v[1] + 1) and (offsets._version, order._version) == (u[0] + 1, u[1] + 1)
    with torch.inference_mode():
        inside = torch.empty((6, 8), device="cuda")
        linear.linear_i8(x, xs, w, ws, out=inside)
    linear.linear_i8(x, xs, w, ws, out=inside)  # has no version to count
    assert torch.equal(inside, out)
    grad = torch.ones(6, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="no gradient"):
        linear.quantize_rows(out, scale=grad)


@pytest.mark.parametrize("kind", KINDS)
def test_the_short_call_is_taken_and_gives_the_same(kind, monkeypatch):
    """pixelbox_amd/_linear_call.so takes the usual calls; without it the same calls go through ctypes"""
    assert linear._load(), "pixelbox_amd/_linear_call.so is not built"
    m, groups, n, k = 100, 3, 40, 64
    x, xs, w, ws, b = grouped_case(kind, m, groups, n, k, 90)
    xf, group = rand((m, k), torch.float32, gen(91)), some_groups(m, groups, 92)

    def everything():
        offsets, order = torch.empty(groups + 1, dtype=torch.int32, device="cuda"), torch.empty(m, dtype=torch.int32, device="cuda")
        c, s = torch.empty((m, k), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")
        linear.group_rows(group, groups, offsets=offsets, order=order)
        linear.quantize_rows(xf, codes=c, scale=s)
        y = linear.linear_grouped(x, w, offsets, rows=order, x_scale=xs, w_scale=ws, bias=b, act="silu", out=torch.zeros((m, n), device="cuda"))
        got = [offsets, order, c, s, y]
        if kind == "i8":
            got.append(linear.linear_i8(x, xs, w[0], ws[0], bias=b[0], out=torch.empty((m, n), dtype=torch.float16, device="cuda")))
        return got

    taken = []

    class Counting:
        def __getattr__(self, name):
            f = getattr(linear._load(), name)

            def call(*a):
                rc = f(*a)
                taken.append((name, rc))
                return rc
            return call

    short = linear._load()
    monkeypatch.setattr(linear, "_load", lambda: short)
    monkeypatch.setattr(linear, "_compiled", Counting())
    first = everything()
    assert all(rc == 0 for _, rc in taken) and len(taken) == len(first) - 2, taken
    monkeypatch.setattr(linear, "_compiled", False)
    assert all(torch.equal(a, b) for a, b in zip(first, everything()))


def test_the_short_call_leaves_the_unusual_alone():
    short = linear._load()
    x, xs, w, ws, b = i8_case(6, 8, 32, 1)
    out = torch.empty((6, 8), device="cuda")
    ok = [x, xs, w, ws, b, 0, out]
    assert short.linear_i8(*ok) == 0
    for i, odd in ((0, x.cpu()), (0, x.float()), (1, xs[:5]), (2, w.t()), (3, None), (4, b.double()), (6, out.t()), (6, out[:, :7]), (0, None)):
        assert short.linear_i8(*ok[:i], odd, *ok[i + 1:]) is None, i
    assert short.linear_i8(x, xs, w, ws, b, 7, out) == -1  # the library's own refusal
    with pytest.raises(capi.PixelboxError):
        linear.linear_i8(x, xs, w, ws, out=x.view(torch.float32)[:, :8].as_strided((6, 8), (8, 1)))  # y over x
