"""pb_embed_heads_device refuses a call before it queues anything, and writes no operand of the caller's."""
import numpy as np
import pytest
import torch

from pixelbox_amd import capi, synth
from pixelbox_amd import weights as W

pytestmark = pytest.mark.gpu

H, N, D, HEADS = 128, 64, 32, 3


def blob(bad=False):
    raw = bytearray(W.synthetic_blob(synth.SEED_WEIGHTS, H, H, 48))
    if bad:  # an activation of 500: outside the domain of the squeeze-excite sums
        at = len(raw) - 4 * sum(int(np.prod(shape)) for _, shape, _ in W.tensor_specs(48))
        for name, shape, _ in W.tensor_specs(48):
            n = int(np.prod(shape))
            if name == "b2.dw.b":
                raw[at:at + 4 * n] = (np.frombuffer(bytes(raw[at:at + 4 * n]), dtype="<f4") + np.float32(500.0)).astype("<f4").tobytes()
            at += 4 * n
    return bytes(raw)


@pytest.fixture(scope="module")
def img():
    return torch.from_numpy(synth.synthetic_images(synth.SEED_IMAGES, 0, N, H, H)).cuda()


def room(i8):
    """weights, scales, bias, heads and outputs in one buffer, a part each"""
    sizes = dict(w=HEADS * D * 1280 * (1 if i8 else 4), scale=HEADS * D * 4, bias=HEADS * D * 4, head=N * 4, f32=N * D * 4, u8=N * D)
    buf, at, pos = torch.zeros(sum(sizes.values()) + 1024, dtype=torch.uint8, device="cuda"), {}, 0
    for name, n in sizes.items():
        at[name] = buf.data_ptr() + pos
        pos += n
    return buf, at


def args(img, at, i8):
    return dict(d_rgb_ptr=img.data_ptr(), n=N, w_type=capi.PB_TYPE_I8 if i8 else capi.PB_TYPE_F32, d_w_ptr=at["w"], heads=HEADS, d=D, d_head_ptr=at["head"],
                d_w_scale_ptr=at["scale"] if i8 else 0, d_bias_ptr=at["bias"], d_out_u8_ptr=at["u8"], d_out_f32_ptr=at["f32"])


@pytest.mark.parametrize("i8", [False, True])
def test_a_refused_call_has_queued_nothing(img, i8):
    emb = capi.Embedder(blob(), max_batch=N)
    s = torch.cuda.Stream()
    emb.set_option(capi.PB_OPT_EMBED_STREAM, s.cuda_stream)
    buf, at = room(i8)
    ok = args(img, at, i8)
    emb.heads_device(**ok)  # the form picks of this batch are made, and the workspace
    refused = [dict(d_out_f32_ptr=at["f32"] + 2), dict(d_head_ptr=at["head"] + 1), dict(d_bias_ptr=at["bias"] + 2),
               dict(d_out_f32_ptr=at["w"] + 64), dict(d_out_f32_ptr=at["bias"]), dict(d_out_f32_ptr=at["head"] - 4 * N * D + 4),
               dict(d_out_u8_ptr=at["w"]), dict(d_out_u8_ptr=at["w"] + HEADS * D * 1280 - 1), dict(d_out_u8_ptr=at["bias"] + HEADS * D * 4 - 1),
               dict(d_out_u8_ptr=at["head"]), dict(d_out_u8_ptr=at["f32"] + 4 * N * D - 1)]
    refused += [dict(d_w_scale_ptr=at["scale"] + 1), dict(d_out_f32_ptr=at["scale"]), dict(d_out_u8_ptr=at["scale"])] if i8 else [dict(d_w_ptr=at["w"] + 2)]
    for change in refused:
        buf.fill_(3)
        torch.cuda.synchronize()
        with pytest.raises(capi.PixelboxError) as e:
            emb.heads_device(**{**ok, **change})
        assert e.value.code == -1, change
        assert s.query(), change  # nothing runs there
        torch.cuda.synchronize()
        assert (buf == 3).all(), change
    emb.heads_device(**ok)
    emb.set_option(capi.PB_OPT_EMBED_STREAM, 0)


def test_a_refused_batch_raises_no_later_error(img):
    emb = capi.Embedder(blob(bad=True), max_batch=N)
    buf, at = room(False)
    ok = args(img, at, False)
    with pytest.raises(capi.PixelboxError) as e:
        emb.heads_device(**ok)
    assert e.value.code == capi.PB_ERR_RANGE
    with pytest.raises(capi.PixelboxError) as e:
        emb.heads_device(**{**ok, "d_w_ptr": at["w"] + 2})
    assert e.value.code == -1
    torch.cuda.synchronize()
    emb.check_range()  # nothing of the refused call
