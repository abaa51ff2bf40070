"""Hash heads on one backbone (pb_embed_features_device, pb_embed_heads_device): the embedder's own path through the grouped and the
8-bit linear layers."""
import numpy as np
import pytest
import torch

import linear_ref as ref
from embed_tol import assert_embeddings_close
from oracle import capi as oracle
from oracle import numpy_oracle as no
from pixelbox_amd import capi, linear, synth
from pixelbox_amd import weights as W

pytestmark = pytest.mark.gpu

H = 64


@pytest.fixture(scope="module")
def blob():
    return W.synthetic_blob(synth.SEED_WEIGHTS, H, H, 48)


@pytest.fixture(scope="module")
def emb(blob):
    return capi.Embedder(blob, max_batch=40)


def images(start, n):
    return torch.from_numpy(synth.synthetic_images(synth.SEED_IMAGES, start, n, H, H)).cuda()


def features(emb, img):
    f = torch.full((img.shape[0], 1280), float("nan"), device="cuda")
    emb.features_device(img.data_ptr(), img.shape[0], f.data_ptr())
    return f


def run(emb, img, head, w, b, scale=None, u8=True, f32=True):
    heads, d = w.shape[:2]
    n = img.shape[0]
    out8 = torch.full((n, d), 7, dtype=torch.uint8, device="cuda")
    out = torch.full((n, d), 9.0, device="cuda")
    emb.heads_device(img.data_ptr(), n, capi.PB_TYPE_I8 if w.dtype == torch.int8 else capi.PB_TYPE_F32, w.data_ptr(), heads, d, head.data_ptr(),
                     0 if scale is None else scale.data_ptr(), 0 if b is None else b.data_ptr(), out8.data_ptr() if u8 else 0, out.data_ptr() if f32 else 0)
    return out8, out


def test_features_make_the_embedding(emb, blob):
    t = W.parse_blob(blob)[3]
    img = images(0, 37)
    f = features(emb, img)
    u8, want = emb.embed(img.cpu().numpy())
    y = np.tanh(f.cpu().double().numpy() @ t["fc.w"].astype(np.float64).T + t["fc.b"].astype(np.float64)).astype(np.float32)
    assert_embeddings_close(y, want)
    for i in (0, 5, 36):  # an image's features do not depend on its batch
        assert torch.equal(features(emb, img[i:i + 1].contiguous())[0], f[i])
    u8_again, want_again = emb.embed(img.cpu().numpy())  # and the ordinary call is what it was
    assert np.array_equal(u8, u8_again) and np.array_equal(want, want_again)


def test_features_of_two_half_batches(emb):
    img = images(50, 40)
    f = features(emb, img)
    emb.set_option(capi.PB_OPT_EMBED_DUAL, 20)
    try:
        assert torch.equal(features(emb, img), f)
        assert torch.equal(features(emb, img), f)
    finally:
        emb.set_option(capi.PB_OPT_EMBED_DUAL, 1024)


def test_the_blobs_own_head_gives_the_embedding(emb, blob):
    t = W.parse_blob(blob)[3]
    img = images(10, 33)
    w = torch.from_numpy(t["fc.w"].copy()).cuda()[None].contiguous()
    b = torch.from_numpy(t["fc.b"].copy()).cuda()[None].contiguous()
    head = torch.zeros(33, dtype=torch.int32, device="cuda")
    u8, f = run(emb, img, head, w, b)
    want = emb.embed(img.cpu().numpy())[1]
    assert_embeddings_close(f.cpu().numpy(), want)
    assert np.array_equal(u8.cpu().numpy(), no.quantize(f.cpu().numpy()))


@pytest.mark.parametrize("n", [1, 2, 17, 40])
@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("heads,d", [(1, 8), (3, 48), (7, 130), (40, 256)])
def test_heads(emb, n, i8, heads, d):
    g = torch.Generator().manual_seed(n * 100 + heads)
    img = images(200, n)
    head = torch.randint(-1, heads + 1, (n,), generator=g, dtype=torch.int32).cuda()
    w = (torch.randn((heads, d, 1280), generator=g) * 0.05).cuda()
    b = torch.randn((heads, d), generator=g).cuda()
    scale = None
    if i8:
        c, s = linear.quantize_rows(w.view(heads * d, 1280))
        w, scale = c.view(heads, d, 1280), s.view(heads, d)
    feat = features(emb, img)
    x, xs = linear.quantize_rows(feat) if i8 else (feat, None)
    offsets, order = ref.group(head, heads)
    want, bound = ref.grouped(x, w, offsets, order, order, b, "tanh", torch.full((n, d), 9.0), xs, scale)
    u8, f = run(emb, img, head, w, b, scale)
    ref.check(f, want, bound)
    has = ((head >= 0) & (head < heads)).cpu()
    assert np.array_equal(u8.cpu()[has].numpy(), no.quantize(f.cpu()[has].numpy()))
    assert (u8.cpu()[~has] == 7).all() and (f.cpu()[~has] == 9.0).all()
    # without the floats: the same bytes from the embedder's own buffer
    u8_only, untouched = run(emb, img, head, w, b, scale, f32=False)
    assert torch.equal(u8_only, u8) and (untouched == 9.0).all()
    _, f_only = run(emb, img, head, w, b, scale, u8=False)
    assert torch.equal(f_only, f)


def test_queued_on_the_callers_stream(emb, blob):
    t = W.parse_blob(blob)[3]
    img = images(70, 24)
    w = torch.from_numpy(t["fc.w"].copy()).cuda()[None].contiguous()
    head = torch.zeros(24, dtype=torch.int32, device="cuda")
    want8, want = run(emb, img, head, w, None)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    emb.set_option(capi.PB_OPT_EMBED_STREAM, s.cuda_stream)
    emb.set_option(capi.PB_OPT_EMBED_ASYNC, 1)
    try:
        with torch.cuda.stream(s):
            for _ in range(3):
                u8, f = run(emb, img, head, w, None)
                assert_later = (u8.clone(), f.clone())  # on the same stream: behind the heads
        s.synchronize()
        emb.check_range()
        assert torch.equal(assert_later[0], want8) and torch.equal(assert_later[1], want)
    finally:
        emb.set_option(capi.PB_OPT_EMBED_ASYNC, 0)
        emb.set_option(capi.PB_OPT_EMBED_STREAM, 0)


def test_refusals(emb):
    img = images(0, 2)
    w, head = torch.zeros((2, 8, 1280), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    o8, o = torch.zeros((2, 8), dtype=torch.uint8, device="cuda"), torch.zeros((2, 8), device="cuda")
    ok = dict(d_rgb_ptr=img.data_ptr(), n=2, w_type=0, d_w_ptr=w.data_ptr(), heads=2, d=8, d_head_ptr=head.data_ptr(), d_out_u8_ptr=o8.data_ptr(),
              d_out_f32_ptr=o.data_ptr())
    emb.heads_device(**ok)
    for change in (dict(n=41), dict(w_type=1), dict(w_type=3), dict(heads=0), dict(heads=1025), dict(d=0), dict(d_out_u8_ptr=0, d_out_f32_ptr=0)):
        with pytest.raises(capi.PixelboxError) as e:
            emb.heads_device(**{**ok, **change})
        assert e.value.code == -1
    with pytest.raises(capi.PixelboxError):
        emb.features_device(img.data_ptr(), 2, o.data_ptr() + 4)
    with pytest.raises(capi.PixelboxError):
        emb.features_device(img.data_ptr(), 41, o.data_ptr())
    emb.heads_device(**{**ok, "n": 0})


def test_buffers_that_overlap_are_refused(emb):
    img = images(0, 4)
    w, head = torch.zeros((2, 8, 1280), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    buf = torch.zeros(64, device="cuda")
    ok = dict(d_rgb_ptr=img.data_ptr(), n=4, w_type=0, d_w_ptr=w.data_ptr(), heads=2, d=8, d_head_ptr=head.data_ptr(), d_out_u8_ptr=buf.data_ptr() + 128,
              d_out_f32_ptr=buf.data_ptr())
    for change in (dict(d_out_u8_ptr=buf.data_ptr() + 127), dict(d_out_u8_ptr=head.data_ptr()), dict(d_out_f32_ptr=head.data_ptr(), d_out_u8_ptr=0),
                   dict(d_out_f32_ptr=w.data_ptr() + 32), dict(d_bias_ptr=buf.data_ptr() + 64)):
        with pytest.raises(capi.PixelboxError) as e:
            emb.heads_device(**{**ok, **change})
        assert e.value.code == -1, change
    with pytest.raises(capi.PixelboxError):
        emb.features_device(img.data_ptr(), 4, img.data_ptr() + 16)
    emb.heads_device(**ok)


def test_heads_of_growing_width(emb):
    """bytes alone: the values go through a buffer of the embedder's that grows with the widest heads so far"""
    g = torch.Generator().manual_seed(8)
    img = images(120, 20)
    head = (torch.arange(20) % 3).to(torch.int32).cuda()
    for d in (16, 200, 24, 1000, 16):
        w = (torch.randn((3, d, 1280), generator=g) * 0.05).cuda()
        only, _ = run(emb, img, head, w, None, f32=False)
        both, _ = run(emb, img, head, w, None)
        assert torch.equal(only, both)


def test_hashes_of_a_head_go_into_its_index(emb):
    """images -> heads -> the index of each collection -> a query answers as the oracle does on those hashes"""
    g = torch.Generator().manual_seed(3)
    n, heads, d = 40, 2, 64
    img = images(300, n)
    head = (torch.arange(n) % heads).to(torch.int32).cuda()
    w = (torch.randn((heads, d, 1280), generator=g) * 0.05).cuda()
    u8, _ = run(emb, img, head, w, None)
    for h in range(heads):
        rows = u8[head == h].contiguous()
        ix = capi.Index(d, 100)
        ids = np.arange(1, rows.shape[0] + 1, dtype=np.int64)
        ix.append_device(ids, rows.data_ptr())
        got, dist, count = ix.search(rows[5:6].cpu().numpy(), 3, 1e3)
        want, want_dist = oracle.scan_topk(rows[5].cpu().numpy(), rows.cpu().numpy(), ids, 3, 1e3)
        assert count[0] == 3 and np.array_equal(got[0], want) and np.array_equal(dist[0], want_dist)
