"""The e4m3 block-scaled path on the GPU: both quantisers bit for bit against the plain form, the product
against float64.

Tolerance of the product: an fp32 sum of n terms, in any order and with each step rounded or cut off, is off by
at most n 2^-23 of the sum of the terms' magnitudes.  A value sums 128 products per block of K, then the blocks,
each times a rounded scale, then a bias: n = 128 + blocks + 4.  The result is rounded to its type once more (half a
step, eps / 2 of its value; for fp16 below 2^-14 half of 2^-24)."""

import ctypes
import math

import numpy as np
import pytest

import e4m3_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f32": 0, "f16": 1, "bf16": 2}


def tdt(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def call(torch, name, *args, stream=None):
    from rembed_b200.embedder import RembedError, library, take_error

    st = torch.cuda.current_stream().cuda_stream if stream is None else stream
    err = ctypes.c_char_p()
    if getattr(library(), name)(*args, st, ctypes.byref(err)) != 0:
        raise RembedError(take_error(err))


def status(torch):
    call(torch, "rg_kernel_status")


def quantize(torch, x, tiles, ldq=None, q_offset=0):
    """x: a 2-D view on the GPU (row stride allowed).  Returns (bytes, scales) as numpy, checking that nothing
    else of the output buffers was written."""
    rows, K = x.shape
    kb = -(-K // 128)
    ldq = ldq or -(-K // 16) * 16
    buf = torch.full((q_offset + rows * ldq + 64,), 0xAB, device="cuda", dtype=torch.uint8)
    name = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[x.dtype]
    if tiles:
        scale = torch.full((-(-rows // 128) + 1, kb), -7.0, device="cuda")
        call(torch, "rg_quantize_tiles_e4m3", x.data_ptr(), DT[name], x.stride(0), rows, K, buf.data_ptr() + q_offset, ldq,
             scale.data_ptr())
        kept = scale[-1:]
        scale = scale[:-1]
    else:
        scale = torch.full((kb, rows + 3), -7.0, device="cuda")
        call(torch, "rg_quantize_rows_e4m3", x.data_ptr(), DT[name], x.stride(0), rows, K, buf.data_ptr() + q_offset, ldq,
             scale.data_ptr(), rows + 3)
        kept = scale[:, rows:]
        scale = scale[:, :rows]
    status(torch)
    assert bool((kept == -7.0).all())
    b = buf.cpu().numpy()
    q = b[q_offset:q_offset + rows * ldq].reshape(rows, ldq)
    assert (b[:q_offset] == 0xAB).all() and (b[q_offset + rows * ldq:] == 0xAB).all() and (q[:, K:] == 0xAB).all()
    return q[:, :K], scale.cpu().numpy()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,K,pad,offset", [
    (1, 1, 0, 0), (1, 128, 0, 0), (7, 127, 0, 0), (8, 129, 3, 0), (9, 300, 0, 1), (128, 256, 8, 0), (129, 1100, 0, 3),
    (300, 768, 4, 0), (17, 2047, 1, 0),
])
def test_quantizers(cuda, tiles, dtype, rows, K, pad, offset):
    """Odd sizes, row strides, and bases that are aligned to nothing but the element."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(rows * K + pad)
    buf = torch.randn((rows * (K + pad) + offset,), device="cuda", generator=g) * 3
    x = buf.to(tdt(torch, dtype))[offset:].view(rows, K + pad)[:, :K]
    q, s = quantize(torch, x, tiles, ldq=K + pad if offset else None, q_offset=offset)
    want_q, want_s = ref.quantize(x.float().cpu().numpy(), 128 if tiles else 1)
    assert np.array_equal(s if tiles else s.T, want_s)
    assert np.array_equal(q, want_q)


@pytest.mark.parametrize("tiles", [False, True])
def test_quantizer_special_values(cuda, tiles):
    """Zeros, subnormals, the largest float32, NaN and infinities: each block for itself."""
    torch = cuda
    x = np.zeros((256, 512), dtype=np.float32)
    x[0, 128:256] = 1e-41  # the block's maximum over 448 would be no normal number
    x[1, 256:384] = np.linspace(-3.4e38, 3.4e38, 128)
    x[130, 5], x[130, 6] = np.nan, 2.0
    x[131, 300], x[131, 301] = -np.inf, 2.0
    q, s = quantize(torch, torch.from_numpy(x).cuda(), tiles)
    want_q, want_s = ref.quantize(x, 128 if tiles else 1)
    got_s = s if tiles else s.T
    assert np.array_equal(got_s, want_s, equal_nan=True)
    nan = np.isnan(ref.decode(want_q))
    assert np.array_equal(np.isnan(ref.decode(q)), nan) and np.array_equal(q[~nan], want_q[~nan])
    with np.errstate(invalid="ignore"):
        back = ref.decode(q) * np.repeat(np.repeat(got_s, 128 if tiles else 1, 0), 128, 1).astype(np.float64)
    assert np.isnan(back[slice(128, 256) if tiles else 130, :128]).all()
    assert np.isnan(back[slice(128, 256) if tiles else 131, 256:384]).all()
    assert np.isfinite(back[:128]).all()


def operands(torch, M, N, K, seed):
    """Quantised operands with unequal scales, as numpy and on the GPU; bytes behind K are e4m3 NaNs."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1)))
    w = rng.standard_normal((N, K)) * 0.05
    (xq, xs), (wq, ws) = ref.quantize(x.astype(np.float32), 1), ref.quantize(w.astype(np.float32), 128)
    out = []
    for q in (xq, wq):
        buf = np.full((q.shape[0], -(-K // 16) * 16 + 16), 0x7F, dtype=np.uint8)
        buf[:, :K] = q
        out.append(torch.from_numpy(buf).cuda())
    return (xq, xs.T, wq, ws), (out[0], torch.from_numpy(np.ascontiguousarray(xs.T)).cuda(), out[1], torch.from_numpy(ws).cuda())


def dense(torch, ops, M, N, K, bias, dtype, ldy=None, offset=0, stream=None, y=None):
    xq, xs, wq, ws = ops
    ldy = ldy or N
    if y is None:
        y = torch.full((offset + M * ldy + 5,), -77.0, device="cuda", dtype=tdt(torch, dtype))
    call(torch, "rg_dense_e4m3", xq.data_ptr(), xq.stride(0), xs.data_ptr(), M, wq.data_ptr(), wq.stride(0),
         ws.data_ptr(), None if bias is None else bias.data_ptr(), y.data_ptr() + offset * y.element_size(), ldy, DT[dtype],
         M, N, K, stream=stream)
    return y


def check(torch, y, host, bias, dtype, M, N, K, ldy, offset):
    want, mag = ref.dense(*host)
    if bias is not None:
        want = want + bias.double().cpu().numpy()
        mag = mag + np.abs(bias.double().cpu().numpy())
    a = y.double().cpu().numpy()
    got = a[offset:offset + M * ldy].reshape(M, ldy)
    assert (a[:offset] == -77).all() and (a[offset + M * ldy:] == -77).all() and (got[:, N:] == -77).all()
    tol = (128 + -(-K // 128) + 4) * 2.0**-23 * mag
    tol = tol + torch.finfo(tdt(torch, dtype)).eps / 2 * (np.abs(want) + tol) + (2.0**-25 if dtype == "f16" else 0)
    err = np.abs(got[:, :N] - want)
    assert (err <= tol).all(), (err / tol).max()


SHAPES = [
    # (M, N, K): one value, one row, the edges of a block and of every tile height and width
    (1, 1, 1), (1, 128, 128), (2, 130, 127), (16, 100, 129), (17, 384, 16), (32, 257, 300), (33, 64, 1100),
    (64, 129, 640), (65, 513, 256), (127, 31, 384), (128, 128, 1152), (129, 1000, 768), (255, 256, 130),
    (256, 512, 512), (300, 2300, 1024), (1003, 1540, 1100), (2500, 640, 256), (4100, 1, 200), (520, 4097, 2000),
]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dense(cuda, M, N, K, dtype):
    torch = cuda
    host, ops = operands(torch, M, N, K, M + N + K)
    bias = torch.randn((N,), device="cuda") if (M + N) % 2 else None
    y = dense(torch, ops, M, N, K, bias, dtype)
    status(torch)
    check(torch, y, host, bias, dtype, M, N, K, N, 0)


@pytest.mark.parametrize("M,N,K", [(3, 200, 256), (40, 333, 384), (700, 600, 512)])
@pytest.mark.parametrize("dtype,pad,offset", [("bf16", 3, 1), ("f16", 8, 8), ("f32", 1, 3), ("f32", 4, 0), ("bf16", 8, 0)])
def test_dense_output_strides(cuda, M, N, K, dtype, pad, offset):
    """Output rows at strides and bases that are aligned to the element alone, or to 16 bytes; nothing else written."""
    torch = cuda
    host, ops = operands(torch, M, N, K, 3)
    y = dense(torch, ops, M, N, K, None, dtype, ldy=N + pad, offset=offset)
    status(torch)
    check(torch, y, host, None, dtype, M, N, K, N + pad, offset)


@pytest.mark.parametrize("M", [5, 700])
def test_dense_nan_stays_in_its_row(cuda, M):
    """A row with a NaN scale, and weights of a tile with an infinite one: NaN there, every other value as without."""
    torch = cuda
    host, ops = operands(torch, M, 400, 384, 5)
    clean = dense(torch, ops, M, 400, 384, None, "f32")
    ops[1][1, 2] = float("nan")
    dirty = dense(torch, ops, M, 400, 384, None, "f32")
    status(torch)
    a, b = (t[:M * 400].view(M, 400).cpu().numpy() for t in (clean, dirty))
    assert np.isnan(b[2]).all()
    assert np.array_equal(np.delete(a, 2, 0), np.delete(b, 2, 0))


def test_dense_fp16_overflow_is_reported(cuda):
    from rembed_b200.embedder import RembedError

    torch = cuda
    _, ops = operands(torch, 4, 128, 128, 9)
    ops[1].fill_(1e6)
    dense(torch, ops, 4, 128, 128, None, "f16")
    with pytest.raises(RembedError, match="fp16"):
        status(torch)
    dense(torch, ops, 4, 128, 128, None, "f32")
    status(torch)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 1024), (37, 1000, 1100), (900, 1152, 768)])
def test_dense_repeats_in_graphs_and_on_streams(cuda, M, N, K):
    """The same bits on every call: on its own, on another stream beside a second call, and replayed from a graph
    with new inputs in the same buffers."""
    torch = cuda
    host, ops = operands(torch, M, N, K, 11)
    _, other = operands(torch, M, N, K, 12)
    first = dense(torch, ops, M, N, K, None, "bf16")
    second = dense(torch, other, M, N, K, None, "bf16")
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = dense(torch, ops, M, N, K, None, "bf16")
    with torch.cuda.stream(s2):
        b = dense(torch, other, M, N, K, None, "bf16")
    torch.cuda.synchronize()
    assert torch.equal(a, first) and torch.equal(b, second)
    held = [t.clone() for t in ops]
    y = torch.full_like(first, -77.0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dense(torch, held, M, N, K, None, "bf16", y=y)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)
    for t, o in zip(held, other):
        t.copy_(o)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, second)
    status(torch)


def test_quantise_then_project(cuda):
    """States quantised on the GPU feed the product directly; the whole is within the operands' rounding."""
    torch = cuda
    M, N, K = 333, 384, 1100
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((M, K), device="cuda", generator=g)
    w = (torch.randn((N, K), device="cuda", generator=g) * 0.02).to(torch.bfloat16)
    ld = -(-K // 16) * 16
    xq, wq = (torch.empty((r, ld), device="cuda", dtype=torch.uint8) for r in (M, N))
    xs, ws = torch.empty((9, M), device="cuda"), torch.empty((3, 9), device="cuda")
    y = torch.empty((M, N), device="cuda")
    call(torch, "rg_quantize_rows_e4m3", x.data_ptr(), 0, K, M, K, xq.data_ptr(), ld, xs.data_ptr(), M)
    call(torch, "rg_quantize_tiles_e4m3", w.data_ptr(), 2, K, N, K, wq.data_ptr(), ld, ws.data_ptr())
    call(torch, "rg_dense_e4m3", xq.data_ptr(), ld, xs.data_ptr(), M, wq.data_ptr(), ld, ws.data_ptr(), None, y.data_ptr(), N, 0, M, N, K)
    status(torch)
    want = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    # each factor is off by at most 2^-4 of itself or, near zero, half of 2^-9 times its block's scale (max / 448)
    tiny = (x.abs().max().double() * 2.0**-10 / 448 * w.double().abs().sum(1)[None] + w.double().abs().max() * 2.0**-10 / 448 * x.double().abs().sum(1)[:, None])
    assert bool(((y.double() - want).abs() <= 2.0**-4 * (2 + 2.0**-4) * mag + 2 * tiny).all())
    rel = float((y.double() - want).norm() / want.norm())
    # independent errors: each factor's relative error is uniform within a step of 2^-3 to 2^-4 of it, rms below 2^-3 / sqrt(12)
    assert rel <= math.sqrt(2) * 2.0**-3 / math.sqrt(12)


@pytest.mark.parametrize("M,N,K", [
    (200, 130, 2048), (300, 100, 2100), (520, 64, 4000), (129, 257, 1500), (1000, 128, 3000),  # few columns, long K
    (70, 9500, 260), (33, 9500, 384), (128, 10001, 129),  # few rows, many columns
    (64, 4736, 1300), (100, 4736, 1100), (40, 2300, 2050),  # as many clusters as SMs have room for, or more
])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_dense_where_the_kernels_meet(cuda, M, N, K, dtype):
    """Few rows through the pairs' kernel, more of them through the one that splits K."""
    torch = cuda
    host, ops = operands(torch, M, N, K, M + N + K)
    bias = torch.randn((N,), device="cuda")
    y = dense(torch, ops, M, N, K, bias, dtype)
    status(torch)
    check(torch, y, host, bias, dtype, M, N, K, N, 0)
