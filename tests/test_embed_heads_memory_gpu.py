"""The room that pb_embed_heads_device takes for its values where the caller wants the bytes alone: that of the images at hand."""
import pytest
import torch

from pixelbox_amd import capi, synth
from pixelbox_amd import weights as W

pytestmark = pytest.mark.gpu

H = 64


def used():
    torch.cuda.synchronize()
    free, total = torch.cuda.mem_get_info()
    return total - free


def test_the_values_take_no_more_than_the_images_at_hand():
    emb = capi.Embedder(W.synthetic_blob(synth.SEED_WEIGHTS, H, H, 48), max_batch=2048)
    img = torch.from_numpy(synth.synthetic_images(synth.SEED_IMAGES, 0, 40, H, H)).cuda()
    head = torch.zeros(40, dtype=torch.int32, device="cuda")
    d = 1 << 18
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn((1, d, 1280), generator=g, device="cuda").mul_(0.05)
    u8, f = torch.zeros((40, d), dtype=torch.uint8, device="cuda"), torch.zeros((40, d), device="cuda")
    # every batch once with the caller's own room for the values, and every comparison: what they load and allocate is there
    for n in (1, 3, 2, 17, 40):
        emb.heads_device(img.data_ptr(), n, 0, w.data_ptr(), 1, d, head.data_ptr(), d_out_u8_ptr=u8.data_ptr(), d_out_f32_ptr=f.data_ptr())
        want = u8.clone()
        assert torch.equal(u8[:n], want[:n]) and (u8[n:] >= 0).all()
    before = used()
    for n, at_most in ((1, 1), (3, 4), (2, 4), (17, 32), (40, 64), (1, 64)):
        u8.zero_()
        emb.heads_device(img.data_ptr(), n, 0, w.data_ptr(), 1, d, head.data_ptr(), d_out_u8_ptr=u8.data_ptr())
        more = used() - before
        assert torch.equal(u8[:n], want[:n]) and (u8[n:] == 0).all()
        assert more <= at_most * d * 4 + (8 << 20), (n, more)  # the smaller ones are given back
