"""64-bit references of the linear layers (pixelbox_amd/linear.py) and the bounds that their results have to keep.

u = 2^-24 is the unit roundoff of f32.  The bounds count roundings:
  * products in f32 (f32, bf16, f16 operands; bf16 and f16 products are exact in f32): k additions in any order are off by at most
    k u sum |x w| (Higham, any order); the matrix cores add several products to a sum at a time and may round each partial sum by a
    whole unit in the last place instead of half of one, so the bound used is 2 k u sum |x w|;
  * 8-bit products are exact sums; (float)sum, * x_scale, * w_scale: 3 u |p|;
  * + bias: u |v|;  both are multiplied by the activation's largest slope (SiLU 1.1, tanh 1);
  * the activation itself: SiLU = v * rcp(1 + exp2(-v log2 e)): the exponent's rounded product is off by |v| log2(e) u and a relative
    (|v| + 1) u of e^-v after that, exp2 and rcp are off by 2 u each, 1 + e^-v, the last product and log2(e)'s own rounding by u
    each: (3 |v| + 8) u |silu(v)| in all (below v = -87.3 the reciprocal may be 0: |v| 2^-126 more); tanh = (1 - e) rcp(1 + e) with e = exp2(-2 |v| log2 e) off by (2 |v| + 2) u of itself, from
    |v| = 0.4 on: the numerator is off by e / (1 - e) (2 |v| + 2) u <= 2.3 u there and rounds by u, the denominator by e / (1 + e) of
    the same <= 0.9 u and rounds by u, rcp 2 u, the product u: 8.2 u; below, the series to v^11: its next term 1 u, the last fused
    step 1 u, what comes before it (a sum below v^3 / 3, 6 % of the result) rounds by less than 1 u in all.  9 u |tanh v| covers both;
  * the result's own rounding: finfo(type).eps / 2 relative, and half of its smallest subnormal.
"""
import torch

U = 2.0 ** -24


def quantize(x: torch.Tensor):
    x = x.detach().cpu()
    top = x.double().abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64)
    bad = ~torch.isfinite(x.double()).all(1)
    scale = torch.clamp((torch.where(bad, torch.ones_like(top), top) / 127.0).float(), min=2.0 ** -126)
    q = x.double() / scale.double()[:, None]
    codes = torch.where(bad[:, None], torch.zeros_like(q), torch.round(q))
    return codes.to(torch.int8), torch.where(bad, torch.full_like(scale, float("nan")), scale)


def act(v: torch.Tensor, name: str) -> torch.Tensor:
    return v * torch.sigmoid(v) if name == "silu" else torch.tanh(v) if name == "tanh" else v


def linear(x, w, bias, name, out_dtype, x_scale=None, w_scale=None):
    """(y, bound) in 64 bits on the CPU; x [m, k], w [n, k]"""
    x64, w64 = x.detach().cpu().double(), w.detach().cpu().double()
    p = x64 @ w64.T
    k = x.shape[1]
    if x.dtype == torch.int8:
        p = p * x_scale.detach().cpu().double()[:, None] * w_scale.detach().cpu().double()
        err = 3 * U * p.abs()
    else:
        err = 2 * k * U * (x64.abs() @ w64.abs().T)
    v = p if bias is None else p + bias.detach().cpu().double()
    err = err + U * v.abs()
    y = act(v, name)
    if name == "silu":
        err = 1.1 * err + (3 * v.abs() + 8) * U * y.abs()
    elif name == "tanh":
        err = err + 9 * U * y.abs()
    info = torch.finfo(out_dtype)
    bound = err * 1.01 + (y.abs() + err) * (info.eps / 2) + info.smallest_normal * info.eps / 2
    return y, bound


def check(got: torch.Tensor, y: torch.Tensor, bound: torch.Tensor, what=""):
    g = got.detach().cpu().double()
    assert g.shape == y.shape, (what, g.shape, y.shape)
    nan = torch.isnan(y)
    assert torch.equal(torch.isnan(g), nan), what
    off = torch.where(nan, torch.zeros_like(g), (g - y).abs() - bound)
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0.0, (what, worst, off.argmax().item())


def group(group: torch.Tensor, groups: int):
    g = group.cpu().long()
    key = torch.where((g >= 0) & (g < groups), g, torch.full_like(g, groups))
    order = torch.tensor(sorted(range(len(key)), key=lambda i: (int(key[i]), i)), dtype=torch.int32)
    offsets = torch.tensor([int((key < i).sum()) for i in range(groups + 1)], dtype=torch.int32)
    return offsets, order


def grouped(x, w, offsets, x_rows, y_rows, bias, name, out, x_scale=None, w_scale=None):
    """(y, bound): `out` (its values before the call) with the listed rows replaced; the bound of the others is 0"""
    y, bound = out.detach().cpu().double().clone(), torch.zeros(out.shape, dtype=torch.float64)
    o = offsets.cpu().tolist()
    for g in range(w.shape[0]):
        at = torch.arange(o[g], o[g + 1])
        if not len(at):
            continue
        xr = x_rows.cpu().long()[at] if x_rows is not None else at
        yr = y_rows.cpu().long()[at] if y_rows is not None else at
        r, b = linear(x.cpu()[xr], w[g], None if bias is None else bias[g], name, out.dtype, None if x_scale is None else x_scale.cpu()[xr],
                      None if w_scale is None else w_scale[g])
        y[yr], bound[yr] = r, b
    return y, bound
