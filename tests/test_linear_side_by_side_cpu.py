"""Column ranges of one wider buffer share no byte: taken as operand and result of one call; ranges that do share bytes are refused (no GPU:
an accepted call ends with the missing device, behind all checks)."""
import pytest

from pixelbox_amd import capi
from test_linear_cpu import P, Q, R, S, grouped, i8, quantize

# rows of 256 bytes: x in the first 128, w, y and codes elsewhere in them
TAKEN = [
    (quantize, dict(x=P, k=32, ldx=64, codes=P + 128, ldc=256)), (quantize, dict(x=P + 128, k=32, ldx=64, codes=P, ldc=256)),
    (quantize, dict(x=P, type=1, k=64, ldx=128, codes=P + 128, ldc=256)), (quantize, dict(x=P, m=1, k=8, ldx=8, codes=P + 32, ldc=8)),
    (quantize, dict(x=P, k=32, ldx=64, scale=P + 128, codes=Q, ldc=32)), (quantize, dict(x=P, k=32, ldx=64, scale=P + 240, codes=Q, ldc=32)),
    (quantize, dict(x=P, k=32, ldx=64, codes=P + 3 * 256 + 128, ldc=32)),  # behind the last row
    (i8, dict(x=P, ldx=256, k=64, n=32, y=P + 128, ldy=64)), (i8, dict(x=P + 128, ldx=256, k=64, n=32, y=P, ldy=64)),
    (i8, dict(w=P, ldw=256, k=64, n=32, x=Q, y=P + 64, ldy=64)), (i8, dict(w=P, ldw=256, k=64, n=32, x=Q, y=P + 64 - 256, ldy=64)),
    (i8, dict(x=P, ldx=256, k=64, n=16, y=P + 192, ldy=64, bias=P + 128, ws=R + (1 << 18))), (i8, dict(y=S, ldy=64, n=32, xs=S + 128, ws=S + 128)),
    (grouped, dict(x=P, ldx=128, k=64, n=32, y=P + 128, ldy=128)), (grouped, dict(w=P, ldw=128, k=64, x=R, n=32, y=P + 128 + 512, ldy=128)),
]
SHARED = [
    (quantize, dict(x=P, k=32, ldx=64, codes=P + 127, ldc=256)), (quantize, dict(x=P, k=32, ldx=64, codes=P + 225, ldc=256)),
    (quantize, dict(x=P + 128, k=32, ldx=64, codes=P + 97, ldc=256)), (quantize, dict(x=P, k=32, ldx=64, codes=P + 128, ldc=255)),
    (quantize, dict(x=P, k=32, ldx=64, scale=P + 244, codes=Q, ldc=32)), (quantize, dict(x=P, k=32, ldx=64, scale=P + 124, codes=Q, ldc=32)),
    (quantize, dict(x=P, k=32, ldx=64, codes=P + 3 * 256 + 127, ldc=32)), (quantize, dict(x=P, m=1, k=8, ldx=8, codes=P + 31, ldc=8)),
    (quantize, dict(x=P, m=1, k=8, ldx=1000, codes=P + 31, ldc=2000)), (quantize, dict(x=P + 4, m=1, k=8, ldx=1000, codes=P - 3, ldc=2000)),
    (i8, dict(x=P, ldx=256, k=64, n=32, y=P + 60, ldy=64)), (i8, dict(x=P, ldx=256, k=64, n=32, y=P + 132, ldy=64)),
    (i8, dict(x=P, ldx=256, k=64, n=33, y=P + 128, ldy=64)), (i8, dict(x=P, ldx=256, k=64, n=32, y=P + 128, ldy=64, bias=P + 64)), (i8, dict(x=P, ldx=256, k=64, n=32, y=P + 64, ldy=65)),
    (i8, dict(x=P, ldx=256, k=64, n=32, y=P + 64 + 512, ldy=64, bias=P + 64 + 512 + 124)), (i8, dict(y=S, ldy=64, n=32, xs=S + 244)),
    (i8, dict(w=P, ldw=256, k=64, n=32, x=Q, y=P - 256 - 64, ldy=64)),
    (grouped, dict(x=P, ldx=128, k=64, n=32, y=P + 126, ldy=128)), (grouped, dict(w=P, ldw=128, k=64, x=R, n=32, y=P + 256 * 100 + 100, ldy=128)),
]


@pytest.mark.skipif(capi.device_count() > 0, reason="the addresses are no memory: only on a box without a GPU")
@pytest.mark.parametrize("call,kw", TAKEN, ids=[f"{c.__name__}-{list(k.items())}" for c, k in TAKEN])
def test_apart(call, kw):
    assert call(**kw) == -2, capi.lib().pb_last_error()  # PB_ERR_HIP: no device, and nothing else


@pytest.mark.parametrize("call,kw", SHARED, ids=[f"{c.__name__}-{list(k.items())}" for c, k in SHARED])
def test_shared_bytes_are_refused(call, kw):
    assert call(**kw) == -1
    assert "overlap" in capi.lib().pb_last_error().decode()
