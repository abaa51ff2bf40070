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


def test_queued_calls_of_growing_width_keep_their_values():
    """calls queued one behind the other, each wider than the last: what is at work with the smaller room is not given another's"""
    emb = capi.Embedder(W.synthetic_blob(synth.SEED_WEIGHTS, H, H, 48), max_batch=64)
    img = torch.from_numpy(synth.synthetic_images(synth.SEED_IMAGES, 500, 40, H, H)).cuda()
    g = torch.Generator().manual_seed(4)
    head = torch.randint(0, 3, (40,), generator=g, dtype=torch.int32).cuda()
    widths = [(5, 40), (64, 17), (300, 40), (1000, 40), (24, 40), (20000, 33), (300, 1)]
    w = {d: (torch.randn((3, d, 1280), generator=g) * 0.05).cuda() for d, _ in widths}
    out = [[torch.zeros((n, d), dtype=torch.uint8, device="cuda") for d, n in widths] for _ in range(4)]
    f32 = [torch.zeros((n, d), device="cuda") for d, n in widths]

    def call(i, u8, f=None):
        d, n = widths[i]
        emb.heads_device(img.data_ptr(), n, 0, w[d].data_ptr(), 3, d, head.data_ptr(), d_out_u8_ptr=u8.data_ptr(), d_out_f32_ptr=0 if f is None else f.data_ptr())

    for i in range(len(widths)):
        call(i, out[0][i], f32[i])  # waits; the values in the caller's room
        call(i, out[1][i])          # waits; in the embedder's, which grows and is given back
    emb = capi.Embedder(W.synthetic_blob(synth.SEED_WEIGHTS, H, H, 48), max_batch=64)
    s = torch.cuda.Stream()
    emb.set_option(capi.PB_OPT_EMBED_STREAM, s.cuda_stream)
    emb.set_option(capi.PB_OPT_EMBED_ASYNC, 1)
    torch.cuda.synchronize()
    for r in (2, 3):
        for i in range(len(widths)):
            call(i, out[r][i])
    s.synchronize()
    emb.check_range()
    emb.set_option(capi.PB_OPT_EMBED_ASYNC, 0)
    emb.set_option(capi.PB_OPT_EMBED_STREAM, 0)
    for r in (1, 2, 3):
        for i in range(len(widths)):
            assert out[r][i].any() and torch.equal(out[r][i], out[0][i]), (r, i)
