"""The e4m3 entry points refuse what they cannot run, with a message and before any CUDA call (no GPU
needed: the pointers are never read), and the plain forms that the GPU tests compare with are right."""

import ctypes

import numpy as np
import pytest

import e4m3_reference as ref

A = 1 << 20  # an aligned address that is never read


def call(name, *args):
    from rembed_b200.embedder import library, take_error

    err = ctypes.c_char_p()
    rc = getattr(library(), name)(*args, None, ctypes.byref(err))
    return None if rc == 0 else take_error(err)


ROWS = dict(x=A, dtype=2, ldx=256, M=4, K=256, q=A, ldq=256, scale=A, ld_scale=4)
TILES = dict(w=A, dtype=0, ldw=256, N=4, K=256, q=A, ldq=256, scale=A)
DENSE = dict(xq=A, ldx=256, xs=A, ld_xs=4, wq=A, ldw=256, ws=A, bias=None, y=A, ldy=8, dtype=2, M=4, N=8, K=256)


@pytest.mark.parametrize("change,word", [
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(dtype=7), "dtype"),
    (dict(K=0), "positive"), (dict(ldx=255), "stride"), (dict(ldq=255), "stride"), (dict(ld_scale=3), "ld_scale"),
    (dict(x=A + 1), "aligned"), (dict(scale=A + 2), "aligned"),
])
def test_quantize_rows_refuses(change, word):
    msg = call("rg_quantize_rows_e4m3", *{**ROWS, **change}.values())
    assert msg and "rg_quantize_rows_e4m3" in msg and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(w=None), "null"), (dict(dtype=-1), "dtype"), (dict(K=-3), "positive"), (dict(ldw=200), "stride"),
    (dict(w=A + 2), "aligned"), (dict(N=65535 * 128 + 1), "over"),
])
def test_quantize_tiles_refuses(change, word):
    msg = call("rg_quantize_tiles_e4m3", *{**TILES, **change}.values())
    assert msg and "rg_quantize_tiles_e4m3" in msg and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(xq=None), "null"), (dict(xs=None), "null"), (dict(wq=None), "null"), (dict(ws=None), "null"),
    (dict(y=None), "null"), (dict(dtype=3), "dtype"), (dict(N=0), "positive"), (dict(K=0), "positive"),
    (dict(ldx=240), "narrower"), (dict(ldw=240), "narrower"), (dict(ldy=7), "narrower"), (dict(ld_xs=3), "narrower"),
    (dict(ldx=264), "16-byte"), (dict(ldw=257), "16-byte"), (dict(xq=A + 8), "16-byte"), (dict(wq=A + 1), "16-byte"),
    (dict(y=A + 1), "aligned"), (dict(bias=A + 2), "aligned"), (dict(M=65535 * 128 + 1, ld_xs=1 << 30), "over"),
])
def test_dense_refuses(change, word):
    msg = call("rg_dense_e4m3", *{**DENSE, **change}.values())
    assert msg and "rg_dense_e4m3" in msg and word in msg, msg


def test_no_rows_is_no_work():
    assert call("rg_quantize_rows_e4m3", *{**ROWS, "M": 0}.values()) is None
    assert call("rg_quantize_tiles_e4m3", *{**TILES, "N": 0}.values()) is None
    assert call("rg_dense_e4m3", *{**DENSE, "M": 0}.values()) is None


def test_reference_codes():
    """Every finite e4m3 byte decodes and encodes to itself; midpoints go to the even code."""
    b = np.array([i for i in range(256) if i & 0x7F != 0x7F], dtype=np.uint8)
    assert np.array_equal(ref.encode(ref.decode(b)), b)
    v = ref.decode(np.arange(0x7F))
    mid = (v[1:] + v[:-1]) / 2
    assert np.array_equal(ref.encode(mid) & 1, np.zeros(0x7E))
    assert ref.decode(0x7E) == 448 and ref.decode(1) == 2.0**-9 and np.isnan(ref.decode(0xFF))
    assert ref.encode(1e9) == 0x7E and ref.encode(-1e9) == 0xFE


def test_reference_product():
    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((5, 300)).astype(np.float32), rng.standard_normal((131, 300)).astype(np.float32)
    (xq, xs), (wq, ws) = ref.quantize(x, 1), ref.quantize(w, 128)
    y, scale = ref.dense(xq, xs.T, wq, ws)
    # each factor is off by at most half a step, 2^-4 of its value (or half the smallest step of its block)
    assert np.all(np.abs(y - x.astype(np.float64) @ w.T.astype(np.float64)) <= (2 * 2.0**-4 + 2.0**-7) * scale + 1e-2)


def test_refuses_what_overflows():
    big, ld = 0x7fffff01, 0x7fffff10
    for name, args in (("rg_quantize_rows_e4m3", {**ROWS, "K": big, "ldx": ld, "ldq": ld}),
                       ("rg_quantize_tiles_e4m3", {**TILES, "K": big, "ldw": ld, "ldq": ld}),
                       ("rg_dense_e4m3", {**DENSE, "K": big, "ldx": ld, "ldw": ld}),
                       ("rg_dense_e4m3", {**DENSE, "N": big, "ldy": ld})):
        msg = call(name, *args.values())
        assert msg and name in msg and "over" in msg, msg
