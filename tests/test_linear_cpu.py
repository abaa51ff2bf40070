"""Refusals of the linear layers (no GPU: nothing is queued, the pointers below are never followed), and the references' own rules."""
import ctypes as C

import pytest
import torch

import linear_ref as ref
from pixelbox_amd import capi, linear

P, Q, R, S = 1 << 20, 2 << 20, 3 << 20, 4 << 20  # addresses that nothing follows


def quantize(**kw):
    a = dict(x=P, type=0, m=4, k=8, ldx=8, codes=Q, ldc=8, scale=R)
    a.update(kw)
    return capi.lib().pb_quantize_rows(0, None, a["x"], a["type"], a["m"], a["k"], a["ldx"], a["codes"], a["ldc"], a["scale"])


def i8(**kw):
    a = dict(x=P, ldx=64, xs=Q, w=R, ldw=64, ws=Q, bias=None, act=0, y=S, yt=0, ldy=32, m=4, n=32, k=64)
    a.update(kw)
    return capi.lib().pb_linear_i8(0, None, a["x"], a["ldx"], a["xs"], a["w"], a["ldw"], a["ws"], a["bias"], a["act"], a["y"], a["yt"], a["ldy"], a["m"],
                                   a["n"], a["k"])


def group(**kw):
    a = dict(group=P, m=100, groups=4, offsets=Q, order=R)
    a.update(kw)
    return capi.lib().pb_group_rows(0, None, a["group"], a["m"], a["groups"], a["offsets"], a["order"])


def grouped(**kw):
    a = dict(type=1, x=P, xt=100, ldx=64, xs=None, w=R, ldw=64, ws=None, bias=None, offsets=Q, groups=4, xr=Q, yr=Q, act=0, y=S, yt=1, ytot=100, ldy=32,
             m=100, n=32, k=64)
    a.update(kw)
    return capi.lib().pb_linear_grouped(0, None, a["type"], a["x"], a["xt"], a["ldx"], a["xs"], a["w"], a["ldw"], a["ws"], a["bias"], a["offsets"],
                                        a["groups"], a["xr"], a["yr"], a["act"], a["y"], a["yt"], a["ytot"], a["ldy"], a["m"], a["n"], a["k"])


REFUSED = [
    (quantize, dict(type=3)), (quantize, dict(type=-1)), (quantize, dict(ldx=7)), (quantize, dict(ldc=7)), (quantize, dict(x=None)), (quantize, dict(codes=None)),
    (quantize, dict(scale=None)), (quantize, dict(x=P + 2)), (quantize, dict(scale=R + 1)), (quantize, dict(codes=P + 100)), (quantize, dict(scale=Q)),
    (quantize, dict(m=1 << 31)), (quantize, dict(ldx=1 << 41)),
    (i8, dict(k=131072, ldx=131072, ldw=131072)), (i8, dict(yt=3)), (i8, dict(act=3)), (i8, dict(act=-1)), (i8, dict(ldx=63)), (i8, dict(ldw=63)), (i8, dict(ldy=31)),
    (i8, dict(x=None)), (i8, dict(w=None)), (i8, dict(y=None)), (i8, dict(xs=None)), (i8, dict(ws=None)), (i8, dict(y=S + 2)), (i8, dict(y=P)),
    (i8, dict(y=R + 64)), (i8, dict(bias=Q + 2)), (i8, dict(m=1 << 31)),
    (group, dict(groups=0)), (group, dict(groups=1025)), (group, dict(group=None)), (group, dict(offsets=None)), (group, dict(order=None)),
    (group, dict(order=P + 4)), (group, dict(offsets=R)), (group, dict(m=1 << 31)), (group, dict(group=P + 2)),
    (grouped, dict(type=4)), (grouped, dict(type=3)), (grouped, dict(yt=3)), (grouped, dict(groups=0)), (grouped, dict(groups=1025)), (grouped, dict(offsets=None)),
    (grouped, dict(offsets=Q + 1)), (grouped, dict(xr=None, xt=99)), (grouped, dict(yr=None, ytot=99)), (grouped, dict(xt=0)), (grouped, dict(ytot=0)),
    (quantize, dict(m=(1 << 31) - 256)), (quantize, dict(m=1 << 30, ldx=1 << 40)), (i8, dict(m=(1 << 31) - 256)), (i8, dict(m=1 << 30, ldy=1 << 40)),
    (group, dict(m=(1 << 31) - 256)), (grouped, dict(m=(1 << 31) - 256, xt=(1 << 31) - 257, ytot=(1 << 31) - 257)), (grouped, dict(ldw=1 << 40, n=1 << 20, ldy=1 << 20)),
    (grouped, dict(xt=(1 << 31) - 256)), (grouped, dict(ytot=(1 << 31) - 256)),
    (i8, dict(xs=S + 64)), (i8, dict(ws=S)), (i8, dict(bias=S + 4)), (grouped, dict(offsets=S + 8)), (grouped, dict(xr=S)), (grouped, dict(yr=S + 64)),
    (grouped, dict(bias=S)),
    (grouped, dict(x=P + 1)), (grouped, dict(y=P + 64)), (grouped, dict(y=R)), (grouped, dict(ldx=63)), (grouped, dict(ldw=10)), (grouped, dict(ldy=1)),
]


@pytest.mark.parametrize("call,kw", REFUSED, ids=[f"{c.__name__}-{list(k.items())}" for c, k in REFUSED])
def test_refused_by_the_library(call, kw):
    assert call(**kw) == -1, capi.lib().pb_last_error()
    assert call.__name__.split("_")[0] in capi.lib().pb_last_error().decode()


@pytest.mark.parametrize("call,kw", [(quantize, dict(m=0, x=None, codes=None, scale=None)), (i8, dict(m=0, x=None, y=None, xs=None)), (i8, dict(n=0, w=None, y=None)),
                                     (grouped, dict(m=0, x=None, offsets=None)), (grouped, dict(n=0, w=None))])
def test_nothing_to_do_is_no_error(call, kw):
    assert call(**kw) == 0


@pytest.mark.skipif(capi.device_count() > 0, reason="only meaningful on a box without a GPU")
@pytest.mark.parametrize("call", [quantize, i8, group, grouped])
def test_no_gpu_is_an_error(call):
    assert call() == -2


def test_torch_forms_refuse_cpu_tensors():
    x = torch.randn(3, 4)
    with pytest.raises(ValueError, match="GPU"):
        linear.quantize_rows(x)
    with pytest.raises(ValueError, match="GPU"):
        linear.linear_i8(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0])
    with pytest.raises(ValueError, match="GPU"):
        linear.group_rows(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="GPU"):
        linear.linear_grouped(x, x[None], torch.zeros(2, dtype=torch.int32))


class _Fake(torch.Tensor):
    """a CPU tensor that says it is on a GPU: what the checks look at ahead of any call into the library"""

    @property
    def device(self):
        return torch.device("cuda", self.__dict__.get("at", 0))

    def get_device(self):
        return self.__dict__.get("at", 0)


def fake(t, at=0):
    f = t.as_subclass(_Fake)
    f.at = at
    return f


def _i8_args():
    return dict(x=fake(torch.zeros((3, 8), dtype=torch.int8)), x_scale=fake(torch.ones(3)), w=fake(torch.zeros((5, 8), dtype=torch.int8)),
                w_scale=fake(torch.ones(5)), out=fake(torch.zeros((3, 5))))


def _grouped_args():
    return dict(x=fake(torch.zeros((3, 8))), w=fake(torch.zeros((2, 5, 8))), offsets=fake(torch.zeros(3, dtype=torch.int32)), out=fake(torch.zeros((3, 5))))


@pytest.mark.parametrize("change,error", [
    (dict(x=fake(torch.zeros((3, 8)))), TypeError), (dict(w=fake(torch.zeros((5, 9), dtype=torch.int8))), ValueError),
    (dict(x_scale=fake(torch.ones(4))), ValueError), (dict(w_scale=fake(torch.ones(5), 1)), ValueError), (dict(bias=fake(torch.ones(4))), ValueError),
    (dict(act="gelu"), ValueError), (dict(out=fake(torch.zeros((3, 5), dtype=torch.int8))), TypeError),
    (dict(out=fake(torch.zeros((5, 3)).t())), ValueError), (dict(out=None, dtype=torch.int8), TypeError),
    (dict(x=fake(torch.zeros(30, dtype=torch.int8).as_strided((3, 8), (4, 1)))), ValueError),
    (dict(w_scale=fake(torch.ones(10)[::2])), ValueError),
])
def test_linear_i8_refuses(change, error):
    with pytest.raises(error):
        linear.linear_i8(**{**_i8_args(), **change})


@pytest.mark.parametrize("change,error", [
    (dict(w=fake(torch.zeros((5, 8)))), ValueError), (dict(w=fake(torch.zeros((2, 5, 8), dtype=torch.float16))), TypeError),
    (dict(offsets=fake(torch.zeros(2, dtype=torch.int32))), ValueError), (dict(offsets=fake(torch.zeros(3, dtype=torch.int64))), TypeError),
    (dict(rows=fake(torch.zeros(3, dtype=torch.int32)), x_rows=fake(torch.zeros(3, dtype=torch.int32))), ValueError),
    (dict(x_rows=fake(torch.zeros(3, dtype=torch.int32)), y_rows=fake(torch.zeros(2, dtype=torch.int32))), ValueError),
    (dict(y_rows=fake(torch.zeros(4, dtype=torch.int32))), ValueError), (dict(x_scale=fake(torch.ones(3))), ValueError),
    (dict(w=fake(torch.zeros((2, 10, 8))[:, ::2])), None), (dict(w=fake(torch.zeros((4, 5, 8))[::2])), ValueError),
    (dict(bias=fake(torch.zeros((4, 5))[::2])), ValueError), (dict(out=fake(torch.zeros((2, 5)))), ValueError),
    (dict(x=fake(torch.zeros((3, 8), dtype=torch.int8)), w=fake(torch.zeros((2, 5, 8), dtype=torch.int8))), ValueError),
    (dict(x=fake(torch.zeros((3, 8), requires_grad=True))), ValueError),
])
def test_linear_grouped_refuses(change, error):
    if error is None:  # every second channel: rows at a stride, groups one behind the other -- a layout that is taken; the library then finds no GPU here
        if capi.device_count() > 0:
            pytest.skip("only meaningful on a box without a GPU")
        error = Exception
    with pytest.raises(error):
        linear.linear_grouped(**{**_grouped_args(), **change})


def test_the_reference_rounds_halves_to_even():
    c, s = ref.quantize(torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5]]))
    assert c.tolist() == [[127, 0, 2, 2, 0, -2]] and s.tolist() == [1.0]
    o, r = ref.group(torch.tensor([2, -1, 0, 2, 9]), 3)
    assert o.tolist() == [0, 1, 1, 3] and r.tolist() == [2, 0, 3, 1, 4]
