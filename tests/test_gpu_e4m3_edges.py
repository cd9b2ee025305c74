"""The e4m3 path where it can go wrong beyond its ordinary shapes: rows of more than 2^31 bytes, values
at and beside ties, rows of y that end within 16 bytes, products of several tiles for each pair of CTAs, splits of K of
every size, infinite scales, special values of 16 bits, and outputs whose rows lie gigabytes apart."""

import numpy as np
import pytest

import e4m3_reference as ref
from test_gpu_e4m3 import DT, call, check, dense, operands, quantize, status, tdt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype,K,rows,pad,offset", [
    ("f32", 2**29 + 300, 1, 0, 0), ("f32", 2**29 + 300, 9, 4, 0), ("f32", 2**29 + 300, 9, 1, 1),
    ("bf16", 2**30 + 300, 1, 0, 0), ("f16", 2**30 + 300, 9, 4, 0), ("bf16", 2**30 + 300, 9, 1, 1),
])
def test_rows_of_more_than_2_31_bytes(cuda, tiles, dtype, K, rows, pad, offset):
    """Columns whose byte offset passes 31 and 32 bits, by every width of load: the blocks at the row's start and end and
    around those columns, against the plain form."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(rows + offset)
    ld, kb = K + pad, -(-K // 128)
    buf = torch.empty((rows * ld + offset,), device="cuda", dtype=tdt(torch, dtype))
    buf.normal_(generator=g)
    x = buf[offset:].view(rows, ld)[:, :K]
    q = torch.full((rows * ld + offset,), 0xAB, device="cuda", dtype=torch.uint8)
    scale = torch.empty((1, kb) if tiles else (kb, rows), device="cuda")
    at = (x.data_ptr(), DT[dtype], ld, rows, K, q.data_ptr() + offset, ld, scale.data_ptr())
    if tiles:
        call(torch, "rg_quantize_tiles_e4m3", *at)
    else:
        call(torch, "rg_quantize_rows_e4m3", *at, rows)
    status(torch)
    got, per = q[offset:].view(rows, ld), 31 - {"f32": 2, "f16": 1, "bf16": 1}[dtype]
    assert bool((got[:, K:] == 0xAB).all()) and bool((q[:offset] == 0xAB).all())
    for col in (0, 2**per - 512, 2**per, K // 128 * 128 - 512, 2**(per - 1)):
        end = min(col + 640, K)
        want_q, want_s = ref.quantize(x[:, col:end].float().cpu().numpy(), 128 if tiles else 1)
        s = scale[:, col // 128:-(-end // 128)] if tiles else scale[col // 128:-(-end // 128)].t()
        assert np.array_equal(s.cpu().numpy(), want_s)
        assert np.array_equal(got[:, col:end].cpu().numpy(), want_q)


def midpoints():
    """Every value halfway between two neighbouring e4m3 values."""
    v = ref.decode(np.arange(0x7F))
    return (v[1:] + v[:-1]) / 2


def tie_rows(rng, rows, bits, exponents, share):
    """fp32 rows of 128 values; `share` of them have one maximum a = 7 m 2^s (m of up to `bits` bits): x = t a / 448 for
    midpoints t, which is an fp32 number where t and m have 24 bits together; every third moved to a neighbour of it."""
    x = np.zeros((rows, 128), dtype=np.float32)
    for r in range(rows):
        if r % share == 0:
            m = int(rng.integers(1, 1 << int(rng.integers(1, bits + 1)))) | 1
            a = np.ldexp(7.0 * m, int(rng.integers(*exponents)))
        t = rng.choice(midpoints(), 128)
        row = (t * (a / 448)).astype(np.float32)
        move = rng.integers(-2, 3, 128) * (rng.random(128) < 1 / 3)
        row = np.where(move < 0, np.nextafter(row, np.float32(0)), np.where(move > 0, np.nextafter(row, np.float32(np.inf)), row))
        row = np.minimum(row, np.float32(a)) * np.where(rng.random(128) < 0.5, -1, 1).astype(np.float32)
        row[int(rng.integers(128))] = a
        x[r] = row
    return x


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("exponents", [(-15, -5), (-100, -80), (80, 104), (-3, 4)])
def test_float32_ties(cuda, tiles, exponents):
    """Quotients that are exact ties, and their neighbours, at ordinary, tiny and huge maxima: the bytes of the exact
    quotient, ties to even."""
    torch = cuda
    x = tie_rows(np.random.default_rng(5), 2048, 20, exponents, 128 if tiles else 1)
    q, s = quantize(torch, torch.from_numpy(x).cuda(), tiles)
    want_q, want_s = ref.quantize(x, 128 if tiles else 1)
    assert np.array_equal(s if tiles else s.T, want_s)
    assert np.array_equal(q, want_q), (q != want_q).sum()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_the_same_values_give_the_same_bytes(cuda, tiles, dtype):
    """16-bit values, ties among them, and the same values as float32."""
    torch = cuda
    x = tie_rows(np.random.default_rng(6), 2048, 6 if dtype == "f16" else 3, (-6, -1), 128 if tiles else 1)
    x = torch.from_numpy(x).cuda().to(tdt(torch, dtype))
    q, s = quantize(torch, x, tiles)
    q32, s32 = quantize(torch, x.float(), tiles)
    assert np.array_equal(s, s32) and np.array_equal(q, q32), (q != q32).sum()


@pytest.mark.parametrize("tiles", [False, True])
def test_ties_over_the_smallest_scale(cuda, tiles):
    """Blocks whose maximum over 448 would be no normal number: x / 2^-126, ties and their neighbours among them."""
    torch = cuda
    rng = np.random.default_rng(7)
    t = midpoints()
    x = rng.choice(t[t <= 300], (512, 128)) * 2.0**-126
    x = (x + rng.integers(-2, 3, x.shape) * 2.0**-149 * (rng.random(x.shape) < 0.5)).astype(np.float32)
    x *= rng.choice([-1, 1], x.shape).astype(np.float32)
    q, s = quantize(torch, torch.from_numpy(x).cuda(), tiles)
    want_q, want_s = ref.quantize(x, 128 if tiles else 1)
    assert (want_s == np.float32(2.0**-126)).all() and np.array_equal(s if tiles else s.T, want_s)
    assert np.array_equal(q, want_q)


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 1])
def test_special_values_of_16_bits(cuda, tiles, dtype, pad):
    """Zeros of both signs, subnormals, the largest values, NaN and infinities in 16 bits: each block for itself."""
    torch = cuda
    big, tiny = (65504.0, 2.0**-24) if dtype == "f16" else (3.38e38, 2.0**-133)
    x = torch.zeros((256, 512 + pad))
    x[:, 1] = -0.0
    x[0, 128:256] = tiny
    x[1, 256:384] = torch.linspace(-big, big, 128)
    x[130, 5], x[130, 6] = float("nan"), 2.0
    x[131, 300], x[131, 301] = -float("inf"), 2.0
    x[132, 400], x[132, 401] = float("inf"), float("nan")
    x = x.to(tdt(torch, dtype)).cuda()[:, :512]
    q, s = quantize(torch, x, tiles)
    want_q, want_s = ref.quantize(x.float().cpu().numpy(), 128 if tiles else 1)
    assert np.array_equal(s if tiles else s.T, want_s, equal_nan=True)
    nan = np.isnan(ref.decode(want_q))
    assert np.array_equal(np.isnan(ref.decode(q)), nan) and np.array_equal(q[~nan], want_q[~nan])


@pytest.mark.parametrize("N", [601, 604, 606, 607, 608, 31])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_columns_behind_the_last_stay(cuda, N, dtype):
    """Rows of y that start on 16-byte boundaries and end between them: what lies behind column N is left alone."""
    torch = cuda
    host, ops = operands(torch, 700, N, 512, N)
    y = dense(torch, ops, 700, N, 512, None, dtype, ldy=N + 16 - N % 8)
    status(torch)
    check(torch, y, host, None, dtype, 700, N, 512, N + 16 - N % 8, 0)


@pytest.mark.parametrize("M,N,K", [(4100, 4500, 100), (4100, 4500, 1100), (4100, 1100, 300), (20000, 300, 260), (5000, 2100, 1100)])
def test_pairs_walk_several_tiles(cuda, M, N, K):
    """Two to five tiles, 256 wide and 128 wide, for each of the 74 pairs of CTAs there are at most: rings, accumulators,
    scales and output boxes carried from one to the next, with one block of K, three and nine.  Outputs by TMA (a
    stride of 16 bytes' multiple) and not."""
    torch = cuda
    assert -(-M // 256) * -(-N // 256) > 74 or -(-M // 256) * -(-N // 128) > 2 * 74
    host, ops = operands(torch, M, N, K, M + K)
    bias = torch.randn((N,), device="cuda")
    for dtype in ("f32", "bf16", "f16"):
        for pad in (3, 4):
            y = dense(torch, ops, M, N, K, bias, dtype, ldy=N + pad)
            status(torch)
            check(torch, y, host, bias, dtype, M, N, K, N + pad, 0)


@pytest.mark.parametrize("M,N,K", [(64, 19200, 1700), (50, 19199, 1700), (64, 12800, 3300), (60, 12700, 3300), (40, 6300, 3300)])
def test_few_rows_and_many_columns(cuda, M, N, K):
    """So many tiles of columns that K is not split, or over two CTAs, or four."""
    torch = cuda
    host, ops = operands(torch, M, N, K, M + N)
    bias = torch.randn((N,), device="cuda")
    for dtype in ("f32", "bf16"):
        y = dense(torch, ops, M, N, K, bias, dtype)
        status(torch)
        check(torch, y, host, bias, dtype, M, N, K, N, 0)


@pytest.mark.parametrize("M", [5, 40, 700])
def test_dense_infinite_weight_scale(cuda, M):
    """One block of 128 x 128 weights with an infinite scale: its columns are infinite or NaN, all others as without."""
    torch = cuda
    _, ops = operands(torch, M, 400, 384, 6)
    clean = dense(torch, ops, M, 400, 384, None, "f32")
    ops[3][1, 2] = float("inf")
    dirty = dense(torch, ops, M, 400, 384, None, "f32")
    status(torch)
    a, b = (t[:M * 400].view(M, 400).cpu().numpy() for t in (clean, dirty))
    assert not np.isfinite(b[:, 128:256]).any()
    assert np.array_equal(np.delete(a, np.s_[128:256], 1), np.delete(b, np.s_[128:256], 1))


@pytest.mark.parametrize("M,K,ldy", [(5, 300, 2**29), (40, 3000, 2**27), (300, 300, 2**24), (300, 300, 2**24 + 1)])
def test_rows_of_y_far_apart(cuda, M, K, ldy):
    """Rows whose offsets pass 2^31 elements and 2^32 bytes, from every kernel and by both ways of writing y."""
    torch = cuda
    N = 136
    host, ops = operands(torch, M, N, K, M)
    y = torch.empty((M * ldy,), device="cuda", dtype=torch.bfloat16)
    rows = y.view(M, ldy)[:, :N + 8]
    rows.fill_(-77.0)
    dense(torch, ops, M, N, K, None, "bf16", ldy=ldy, y=y)
    status(torch)
    check(torch, torch.cat([rows.reshape(-1), rows.new_full((5,), -77.0)]), host, None, "bf16", M, N, K, N + 8, 0)
