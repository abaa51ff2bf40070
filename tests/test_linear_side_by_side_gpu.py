"""Features, codes and hashes side by side in the rows of one wider tensor."""
import pytest
import torch

import linear_ref as ref
from pixelbox_amd import capi, linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [5, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_layer_writes_beside_its_input(m, dtype):
    k, n = 200, 72
    g = torch.Generator().manual_seed(m)
    wide = torch.full((m, 400), 5.0, dtype=dtype, device="cuda")
    wide[:, 8:8 + k] = torch.randn((m, k), generator=g).to(dtype).cuda()
    w, b = (torch.randn((1, n, k), generator=g) * 0.1).to(dtype).cuda(), torch.randn((1, n), generator=g).cuda()
    offsets = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    before = wide.clone()
    want, bound = ref.linear(before[:, 8:8 + k], w[0], b[0], "tanh", dtype)
    for at in (208, 8 + k, 400 - n):
        wide.copy_(before)
        out = linear.linear_grouped(wide[:, 8:8 + k], w, offsets, bias=b, act="tanh", out=wide[:, at:at + n])
        ref.check(out, want, bound, at)
        left = torch.ones(400, dtype=torch.bool)
        left[at:at + n] = False
        assert torch.equal(wide[:, left], before[:, left])
    for at in (207, 0, 9, 150):  # into the input
        with pytest.raises(capi.PixelboxError, match="overlaps"):
            linear.linear_grouped(wide[:, 8:8 + k], w, offsets, bias=b, out=wide[:, at:at + n])


def test_codes_beside_their_rows():
    m, k = 300, 130
    wide = torch.zeros((m, 4 * k + 144 + 4 * 5), dtype=torch.uint8, device="cuda")  # k floats, k codes, then what is left alone
    pitch = wide.shape[1]
    x = wide.view(torch.float32)[:, :k]
    x.copy_(torch.randn((m, k), generator=torch.Generator().manual_seed(1)).cuda())
    wide[:, 5 * k:] = 9
    codes = wide.view(torch.int8)[:, 4 * k:5 * k]
    assert x.stride(0) * 4 == codes.stride(0) == pitch
    want, scale = linear.quantize_rows(x.contiguous())
    got, s = linear.quantize_rows(x, codes=codes)
    assert torch.equal(got, want) and torch.equal(s, scale) and (wide[:, 5 * k:] == 9).all()
    # and the 8-bit product of those codes, back into the same rows
    w, ws = linear.quantize_rows(torch.randn((4, k), generator=torch.Generator().manual_seed(2)).cuda())
    out = wide.view(torch.float32)[:, 166:170]
    y = linear.linear_i8(codes, s, w, ws, out=out)
    assert torch.equal(y, linear.linear_i8(want, scale, w, ws)) and torch.equal(codes, want)
