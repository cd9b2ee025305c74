"""rg_cross_attention refuses what it cannot run, with a message and before any CUDA call (no GPU needed: the
pointers are never read)."""

import ctypes

import pytest

A = 1 << 20  # an aligned address that is never read
ARGS = dict(q=A, k=A, v=A, ldq=128, ldk=128, ldv=128, cu_q=A, kv_begin=A, kv_len=A, nseq=2, Tq=10, Tk=20, max_q=5,
            max_kv=20, heads=2, kv_heads=1, head_dim=64, scale=0.125, dtype=2, out=A, ldo=128)


def call(**change):
    from rembed_b200.embedder import library, take_error

    err = ctypes.c_char_p()
    rc = library().rg_cross_attention(*{**ARGS, **change}.values(), None, ctypes.byref(err))
    return None if rc == 0 else take_error(err)


@pytest.mark.parametrize("change,word", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(cu_q=None), "null"),
    (dict(kv_begin=None), "null"), (dict(kv_len=None), "null"), (dict(out=None), "null"), (dict(dtype=0), "dtype"),
    (dict(head_dim=96), "head dim"), (dict(heads=3, kv_heads=2), "multiple"), (dict(kv_heads=0), "multiple"),
    (dict(ldq=120), "narrower"), (dict(ldk=56), "narrower"), (dict(ldv=56), "narrower"), (dict(ldo=64), "narrower"),
    (dict(ldq=132), "16-byte"), (dict(ldo=129), "16-byte"), (dict(k=A + 8), "16-byte"), (dict(out=A + 2), "16-byte"),
    (dict(cu_q=A + 1), "aligned"), (dict(Tk=0), "positive"), (dict(max_q=0), "positive"), (dict(max_kv=-1), "positive"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(nseq=1 << 30, Tq=1 << 30, max_q=1 << 30), "too many"),
])
def test_refuses(change, word):
    msg = call(**change)
    assert msg and "rg_cross_attention" in msg and word in msg, msg


def test_no_queries_is_no_work():
    assert call(nseq=0) is None
    assert call(Tq=0) is None


@pytest.mark.parametrize("change,word", [
    (dict(scale=2.5e38), "scale"),  # times log2(e) it is infinite in fp32
    (dict(Tq=0x7fffff01), "over"), (dict(Tk=0x7fffff01), "over"),
])
def test_refuses_what_overflows(change, word):
    msg = call(**change)
    assert msg and "rg_cross_attention" in msg and word in msg, msg
