"""Hash heads (pb_embed_heads_device): an image's hash is the same bits in every batch, as the embedder's own is."""
import numpy as np
import pytest
import torch

from pixelbox_amd import capi, linear, synth
from pixelbox_amd import weights as W

pytestmark = pytest.mark.gpu

H = 64


@pytest.fixture(scope="module")
def images():
    return torch.from_numpy(synth.synthetic_images(synth.SEED_IMAGES, 0, 2048, H, H)).cuda()


@pytest.fixture(scope="module")
def emb():
    return capi.Embedder(W.synthetic_blob(synth.SEED_WEIGHTS, H, H, 48), max_batch=2048)


def run(emb, img, head, w, b, scale=None):
    heads, d = w.shape[:2]
    n = img.shape[0]
    u8 = torch.full((n, d), 7, dtype=torch.uint8, device="cuda")
    f = torch.full((n, d), 9.0, device="cuda")
    emb.heads_device(img.data_ptr(), n, capi.PB_TYPE_I8 if scale is not None else capi.PB_TYPE_F32, w.data_ptr(), heads, d, head.data_ptr(),
                     0 if scale is None else scale.data_ptr(), b.data_ptr(), u8.data_ptr(), f.data_ptr())
    return u8, f


# widths at which 2048, 512, 40 and 1 images go through different kernel forms; an odd one
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads,d", [(8, 256), (1, 256), (3, 1001), (40, 64)])
def test_a_hash_does_not_depend_on_its_batch(emb, images, heads, d, i8):
    g = torch.Generator().manual_seed(heads * 1000 + d)
    w = (torch.randn((heads, d, 1280), generator=g) * 0.05).cuda()
    b = (torch.randn((heads, d), generator=g) * 0.1).cuda()
    scale = None
    if i8:
        c, s = linear.quantize_rows(w.view(heads * d, 1280))
        w, scale = c.view(heads, d, 1280), s.view(heads, d)
    head = torch.randint(-1, heads, (2048,), generator=g, dtype=torch.int32).cuda()
    u8, f = run(emb, images, head, w, b, scale)
    has = head >= 0
    assert torch.isfinite(f[has]).all() and f[has].abs().max() <= 1.0
    for start, n in ((0, 1), (2047, 1), (100, 2), (7, 40), (300, 128), (0, 256), (512, 512), (3, 1024), (0, 2000)):
        u8n, fn = run(emb, images[start:start + n].contiguous(), head[start:start + n].contiguous(), w, b, scale)
        assert torch.equal(fn.view(torch.int32), f[start:start + n].view(torch.int32)), (start, n)
        assert torch.equal(u8n, u8[start:start + n]), (start, n)


def test_a_hash_does_not_depend_on_the_other_heads(emb, images):
    """the same weights as the only head and as one of many, at the same and at another width"""
    g = torch.Generator().manual_seed(9)
    w, b = (torch.randn((40, 320, 1280), generator=g) * 0.05).cuda(), torch.randn((40, 320), generator=g).cuda()
    head = torch.randint(0, 40, (900,), generator=g, dtype=torch.int32).cuda()
    img = images[:900].contiguous()
    u8, f = run(emb, img, head, w, b)
    for h in (0, 13, 39):
        at = (head == h).nonzero().squeeze(1)
        one = torch.zeros(at.numel(), dtype=torch.int32, device="cuda")
        for d in (320, 77):
            u8h, fh = run(emb, img[at].contiguous(), one, w[h:h + 1, :d].contiguous(), b[h:h + 1, :d].contiguous())
            assert torch.equal(fh.view(torch.int32), f[at, :d].view(torch.int32)) and torch.equal(u8h, u8[at, :d]), (h, d)


def test_more_channels_than_one_launch_has_threads_for():
    """8192 images of 2^20 channels: several launches, each with its own channels"""
    d, n = 1 << 20, 8192
    emb = capi.Embedder(W.synthetic_blob(synth.SEED_WEIGHTS, 32, 32, 8), max_batch=n)
    img = torch.randint(0, 256, (n, 32, 32, 3), generator=torch.Generator().manual_seed(1), dtype=torch.uint8).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn((1, d, 1280), generator=g, device="cuda").mul_(0.05)
    b = torch.randn((1, d), generator=g, device="cuda")
    head = torch.zeros(n, dtype=torch.int32, device="cuda")
    head[5] = -1
    u8, f = run(emb, img, head, w, b)
    assert (u8[5] == 7).all() and (f[5] == 9.0).all()
    for c in (0, 77, d // 2 - 31, d - 64):
        u8c, fc = run(emb, img, head, w[:, c:c + 64].contiguous(), b[:, c:c + 64].contiguous())
        assert torch.equal(fc.view(torch.int32), f[:, c:c + 64].view(torch.int32)) and torch.equal(u8c, u8[:, c:c + 64]), c
    q = f[:50, :1000].cpu().numpy()
    assert np.isfinite(q).all()
