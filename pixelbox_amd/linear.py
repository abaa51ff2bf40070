"""Linear layers on torch tensors: 8-bit products with a scale per row and channel, and products grouped by expert.

The tensor-facing form of pb_quantize_rows, pb_linear_i8, pb_group_rows and pb_linear_grouped (include/pixelbox_hip.h): shapes, types,
strides and devices are checked here, the work is queued on the tensors' device on torch's current stream, and nothing waits for it.

    w_codes, w_scale = quantize_rows(weight)                     # once: weight [n, k] -> codes and a scale per channel
    codes, scale = quantize_rows(features)                       # per batch
    y = linear_i8(codes, scale, w_codes, w_scale, bias, act="tanh")

    offsets, order = group_rows(head_of_image, heads)            # images of a batch -> rows in the order of their heads
    y = linear_grouped(features, weights, offsets, rows=order, bias=bias, act="tanh")   # weights [heads, n, k]

Rows may have any stride >= their length (a slice of a wider tensor), the last axis is contiguous; an output overlaps no other
tensor of its call.  Products have no derivative, backward or forward: an operand that requires a gradient or carries a tangent is
refused, and an output that a backward pass has saved is counted as written.  Negated views are refused too.
"""
from __future__ import annotations

import ctypes as C
import sysconfig
import warnings

import torch
from torch.autograd import forward_ad

from . import capi

_TYPES = {torch.float32: capi.PB_TYPE_F32, torch.bfloat16: capi.PB_TYPE_BF16, torch.float16: capi.PB_TYPE_F16, torch.int8: capi.PB_TYPE_I8}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ACTS = {"none": capi.PB_ACT_NONE, "silu": capi.PB_ACT_SILU, "tanh": capi.PB_ACT_TANH}


# the current stream's handle without making a Stream object: 0.1 us a call instead of 1.7
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(index: int) -> int:
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _device(t: torch.Tensor, name: str) -> int:
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} is on {t.device}: the operators run on a GPU")
    return index


# One call of these operators is a kernel of a few microseconds; checks from Python and ctypes take as long again.  _linear_call (csrc/
# pb_linear_call.cpp, built beside the library) looks at the usual call -- plain contiguous tensors of the right types, shapes and device -- and
# makes it; it answers None for any other, which is then checked here, name by name, and made through ctypes.
_compiled = None


def _usable(module):
    """the module if it was built for the running torch and Python, whose layouts it has compiled in; else False"""
    here = f"torch {torch.__version__} {sysconfig.get_config_var('SOABI')}"
    built = getattr(module, "built_for", "an unknown torch")
    if built == here:
        return module
    warnings.warn(f"pixelbox_amd: _linear_call.so was built for {built}, this is {here}: calls take the longer way until it is built again")
    return False


def _load():
    global _compiled
    L = capi.lib()
    try:
        from . import _linear_call
    except ImportError:  # not built: the calls below do the same
        _compiled = False
    else:
        _compiled = _usable(_linear_call)
    if _compiled:
        _compiled.bind(*(C.cast(f, C.c_void_p).value for f in (L.pb_quantize_rows, L.pb_linear_i8, L.pb_group_rows, L.pb_linear_grouped)))
    return _compiled


def _check(t: torch.Tensor, name: str, shape: tuple, dtypes: tuple, index: int) -> None:
    """dtype, device, shape (None: any length), a contiguous last axis and values that are what lies in memory"""
    if t.is_neg():  # a view whose values are the memory's with the other sign
        raise ValueError(f"{name} is a negated view (resolve_neg() gives a tensor of its own)")
    if t.dtype in dtypes and t.get_device() == index and t.shape == shape and t.is_contiguous():
        return
    if t.dtype not in dtypes:
        raise TypeError(f"{name} is {t.dtype}, not {' or '.join(str(d) for d in dtypes)}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, x is on GPU {index}")
    if t.dim() != len(shape) or any(want is not None and have != want for have, want in zip(t.shape, shape)):
        raise ValueError(f"{name} has the shape {tuple(t.shape)}, not {shape}")
    if t.numel() and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last axis is not contiguous")


def _ld(t: torch.Tensor, name: str) -> int:
    """distance between the rows of a 2-d tensor"""
    n = t.shape[1]
    if t.is_contiguous() or t.shape[0] <= 1:
        return n
    ld = t.stride(0)
    if ld < n:
        raise ValueError(f"{name}: rows overlap (a stride of {ld} for {n} values)")
    return ld


def _no_grad(*tensors) -> None:
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if grad and t.requires_grad:
            raise ValueError("these products have no gradient: an operand requires one (detach it, or call under torch.no_grad())")
        if forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("these products have no derivative: an operand has a tangent (torch.autograd.forward_ad.unpack_dual gives its values alone)")


def _written(*tensors) -> None:
    """the caller's tensors that a call writes: a backward pass that saved their old values is to say so"""
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _act(act: str) -> int:
    if act not in _ACTS:
        raise ValueError(f"act is {act!r}, not one of {', '.join(_ACTS)}")
    return _ACTS[act]


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _call(rc: int) -> None:
    if rc != capi.PB_OK:
        capi._check(rc)


def quantize_rows(x: torch.Tensor, codes: torch.Tensor | None = None, scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [m, k] (f32, bf16, f16) -> (codes int8 [m, k], scale f32 [m]): scale = max(max |x| / 127, 2^-126) of each row, codes rounded to the
    nearest, halves to even.  A row with an infinity or a NaN has scale NaN and codes 0."""
    short = _load() if _compiled is None else _compiled
    if short and codes is not None and scale is not None:
        rc = short.quantize_rows(x, codes, scale)
        if rc == 0:
            return codes, scale
        if rc is not None:
            _call(rc)
    dev = _device(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x has the shape {tuple(x.shape)}, not (rows, values)")
    m, k = x.shape
    _check(x, "x", (m, k), _FLOATS, dev)
    _no_grad(x, scale)
    if codes is None:
        codes = torch.empty((m, k), dtype=torch.int8, device=x.device)
    else:
        _check(codes, "codes", (m, k), (torch.int8,), dev)
    if scale is None:
        scale = torch.empty((m,), dtype=torch.float32, device=x.device)
    else:
        _check(scale, "scale", (m,), (torch.float32,), dev)
    ldx, ldc = _ld(x, "x"), _ld(codes, "codes")
    _written(codes, scale)
    _call(capi.lib().pb_quantize_rows(dev, _stream(dev), x.data_ptr(), _TYPES[x.dtype], m, k, ldx, codes.data_ptr(), ldc, scale.data_ptr()))
    return codes, scale


def linear_i8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None, act: str = "none",
              dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """act((x w^T) * x_scale * w_scale + bias): x int8 [m, k], w int8 [n, k], x_scale f32 [m], w_scale f32 [n], bias f32 [n].  The result has
    `dtype`, or out's."""
    code = _act(act)
    short = _load() if _compiled is None else _compiled
    if short and out is not None:
        rc = short.linear_i8(x, x_scale, w, w_scale, bias, code, out)
        if rc == 0:
            return out
        if rc is not None:
            _call(rc)
    dev = _device(x, "x")
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError(f"x and w have the shapes {tuple(x.shape)} and {tuple(w.shape)}, not (m, k) and (n, k)")
    m, k = x.shape
    n = w.shape[0]
    _check(x, "x", (m, k), (torch.int8,), dev)
    _check(w, "w", (n, k), (torch.int8,), dev)
    _check(x_scale, "x_scale", (m,), (torch.float32,), dev)
    _check(w_scale, "w_scale", (n,), (torch.float32,), dev)
    if bias is not None:
        _check(bias, "bias", (n,), (torch.float32,), dev)
    _no_grad(x_scale, w_scale, bias, out)
    if out is None:
        if dtype not in _FLOATS:
            raise TypeError(f"dtype is {dtype}, not one of {', '.join(str(d) for d in _FLOATS)}")
        out = torch.empty((m, n), dtype=dtype, device=x.device)
    else:
        _check(out, "out", (m, n), _FLOATS, dev)
    ldx, ldw, ldy = _ld(x, "x"), _ld(w, "w"), _ld(out, "out")
    _written(out)
    _call(capi.lib().pb_linear_i8(dev, _stream(dev), x.data_ptr(), ldx, x_scale.data_ptr(), w.data_ptr(), ldw, w_scale.data_ptr(), _ptr(bias), code,
                                  out.data_ptr(), _TYPES[out.dtype], ldy, m, n, k))
    return out


def group_rows(group: torch.Tensor, groups: int, offsets: torch.Tensor | None = None, order: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """group int32 [m] -> (offsets int32 [groups + 1], order int32 [m]): group g's rows are order[offsets[g] : offsets[g + 1]], ascending.  Rows with a
    group outside [0, groups) come last, behind offsets[groups]."""
    short = _load() if _compiled is None else _compiled
    if short and offsets is not None and order is not None:
        rc = short.group_rows(group, groups, offsets, order)
        if rc == 0:
            return offsets, order
        if rc is not None:
            _call(rc)
    dev = _device(group, "group")
    if group.dim() != 1:
        raise ValueError(f"group has the shape {tuple(group.shape)}, not (rows,)")
    m = group.shape[0]
    _check(group, "group", (m,), (torch.int32,), dev)
    if not 1 <= groups <= capi.PB_MAX_GROUPS:
        raise ValueError(f"groups is {groups}, not 1 .. {capi.PB_MAX_GROUPS}")
    if offsets is None:
        offsets = torch.empty((groups + 1,), dtype=torch.int32, device=group.device)
    else:
        _check(offsets, "offsets", (groups + 1,), (torch.int32,), dev)
    if order is None:
        order = torch.empty((m,), dtype=torch.int32, device=group.device)
    else:
        _check(order, "order", (m,), (torch.int32,), dev)
    _written(offsets, order)
    _call(capi.lib().pb_group_rows(dev, _stream(dev), group.data_ptr(), m, groups, offsets.data_ptr(), order.data_ptr()))
    return offsets, order


def linear_grouped(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, rows: torch.Tensor | None = None, x_rows: torch.Tensor | None = None,
                   y_rows: torch.Tensor | None = None, x_scale: torch.Tensor | None = None, w_scale: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, act: str = "none", dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[yr(r)] = act(x[xr(r)] w[g]^T (* x_scale[xr(r)] * w_scale[g]) + bias[g]) for every group g and r in [offsets[g], offsets[g + 1]).

    x [rows of x, k] (f32, bf16, f16; int8 with x_scale [rows of x] and w_scale [groups, n]), w [groups, n, k], bias f32 [groups, n], offsets int32
    [groups + 1].  x_rows and y_rows (int32 [m], `rows` for both) name the row of x that is read and the row of out that is written at each place r;
    without them it is r itself.  Rows of out that no place names are left as they are: zero where out is made here (m rows, or as many as x
    has if that is more and y_rows is given)."""
    code = _act(act)
    if rows is not None:
        if x_rows is not None or y_rows is not None:
            raise ValueError("rows stands for x_rows and y_rows: give one or the other")
        x_rows = y_rows = rows
    short = _load() if _compiled is None else _compiled
    if short and out is not None:
        rc = short.linear_grouped(x, w, offsets, x_rows, y_rows, x_scale, w_scale, bias, code, out)
        if rc == 0:
            return out
        if rc is not None:
            _call(rc)
    dev = _device(x, "x")
    if x.dim() != 2 or w.dim() != 3:
        raise ValueError(f"x and w have the shapes {tuple(x.shape)} and {tuple(w.shape)}, not (rows, k) and (groups, n, k)")
    x_total, k = x.shape
    groups, n, _ = w.shape
    _check(x, "x", (x_total, k), _FLOATS + (torch.int8,), dev)
    _check(w, "w", (groups, n, k), (x.dtype,), dev)
    if not 1 <= groups <= capi.PB_MAX_GROUPS:
        raise ValueError(f"w has {groups} groups, not 1 .. {capi.PB_MAX_GROUPS}")
    ldw = k
    if not w.is_contiguous():
        ldw = w.stride(1) if n > 1 else w.stride(0) if n == 1 and groups > 1 else k
        if ldw < k or (groups > 1 and n > 0 and w.stride(0) != n * ldw):
            raise ValueError("w: the groups' weights do not follow one another row by row")
    _check(offsets, "offsets", (groups + 1,), (torch.int32,), dev)
    m = x_total
    if x_rows is not None:
        m = x_rows.numel()
        _check(x_rows, "x_rows", (m,), (torch.int32,), dev)
    if y_rows is not None and y_rows is not x_rows:
        m = y_rows.numel()
        _check(y_rows, "y_rows", (m,), (torch.int32,), dev)
        if x_rows is not None and x_rows.shape[0] != m:
            raise ValueError(f"x_rows and y_rows differ in length: {x_rows.shape[0]}, {m}")
    if x_rows is None and m > x_total:
        raise ValueError(f"y_rows lists {m} rows, x has {x_total}")
    i8 = x.dtype == torch.int8
    if i8:
        if x_scale is None or w_scale is None:
            raise ValueError("8-bit operands need x_scale and w_scale")
        _check(x_scale, "x_scale", (x_total,), (torch.float32,), dev)
        _check(w_scale, "w_scale", (groups, n), (torch.float32,), dev)
    elif x_scale is not None or w_scale is not None:
        raise ValueError("scales are for 8-bit operands")
    if bias is not None:
        _check(bias, "bias", (groups, n), (torch.float32,), dev)
    for t, name in ((w_scale, "w_scale"), (bias, "bias")):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{name}: the groups' rows do not follow one another")
    _no_grad(x, w, x_scale, w_scale, bias, out)
    if out is None:
        dtype = dtype or (torch.float32 if i8 else x.dtype)
        if dtype not in _FLOATS:
            raise TypeError(f"dtype is {dtype}, not one of {', '.join(str(d) for d in _FLOATS)}")
        out = torch.zeros((m if y_rows is None else max(m, x_total), n), dtype=dtype, device=x.device)
    else:
        _check(out, "out", (out.shape[0] if out.dim() else 0, n), _FLOATS, dev)
        if y_rows is None and out.shape[0] < m:
            raise ValueError(f"out has {out.shape[0]} rows, {m} may be written")
    if m == 0 or n == 0 or (out.shape[0] == 0 and y_rows is not None) or x_total == 0:
        return out
    ldx, ldy = _ld(x, "x"), _ld(out, "out")
    _written(out)
    _call(capi.lib().pb_linear_grouped(dev, _stream(dev), _TYPES[x.dtype], x.data_ptr(), x_total, ldx, _ptr(x_scale), w.data_ptr(), ldw,
                                       _ptr(w_scale), _ptr(bias), offsets.data_ptr(), groups, _ptr(x_rows), _ptr(y_rows), code, out.data_ptr(),
                                       _TYPES[out.dtype], out.shape[0], ldy, m, n, k))
    return out
