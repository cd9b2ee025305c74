"""rg_cross_attention against a float64 softmax of the same 16-bit inputs.

Tolerance, per output value, with u half a step of the type (2^-8 bf16, 2^-11 fp16) and A = sum_j p_j |v_j| over
the exact probabilities p: each probability enters the product rounded (u A) and the result is rounded (u |o|).  A
score is an fp32 sum of D products, off by at most D 2^-23 scale sum |q| |k|, and passes through two roundings and a
hardware exponential (2^-22 and 2^-23 of the score's size): with d that error at its largest over the row, the weights
move by a factor within exp(+-2 d), so the output by 2 d A, doubled for its second order.  A share of the exponentials
is a polynomial (2.7e-6, below 2^-18 of its value): 2^-17 A.  The products' and the
sum's fp32 additions add (keys + 16) 2^-23 A, and in fp16 a probability below 2^-14 keeps 2^-25 absolute:
2^-25 sum |v|."""

import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

DT = {"f16": 1, "bf16": 2}


def call(torch, *args, stream=None):
    from rembed_b200.embedder import RembedError, library, take_error

    st = torch.cuda.current_stream().cuda_stream if stream is None else stream
    err = ctypes.c_char_p()
    if library().rg_cross_attention(*args, st, ctypes.byref(err)) != 0:
        raise RembedError(take_error(err))


def status(torch):
    from rembed_b200.embedder import RembedError, library, take_error

    err = ctypes.c_char_p()
    if library().rg_kernel_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(err)) != 0:
        raise RembedError(take_error(err))


class Batch:
    """Query sequences of lengths ql over texts of lengths kl; `padded`: texts at a common stride, NaN behind their
    ends (and before the first), `shared`: every query sequence reads the first text."""

    def __init__(self, torch, ql, kl, heads, kv_heads, dim, dtype, seed, padded=False, shared=False, pad_q=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        tdt = {"f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        self.torch, self.ql, self.kl, self.heads, self.kv_heads, self.dim, self.dtype = torch, ql, kl, heads, kv_heads, dim, dtype
        if shared:
            self.kl = kl = [kl[0]] * len(ql)
        self.Tq = sum(ql) + pad_q  # rows behind the last sequence
        self.cu = [sum(ql[:i]) for i in range(len(ql) + 1)]
        stride = max(kl) + 5
        self.begin = [0 if shared else 3 + i * stride if padded else sum(kl[:i]) for i in range(len(kl))]
        self.Tk = max(1, (3 + len(kl) * stride) if padded else (kl[0] if shared else sum(kl)))
        kvd = kv_heads * dim
        self.q = (1.5 * torch.randn((self.Tq, heads * dim + 8), device="cuda", generator=g)).to(tdt)
        self.kv = torch.randn((self.Tk, 2 * kvd), device="cuda", generator=g).to(tdt)
        if padded:
            keep = torch.zeros(self.Tk, dtype=torch.bool)
            for b, n in zip(self.begin, kl):
                keep[b:b + n] = True
            self.kv[~keep.cuda()] = float("nan")
        self.out = torch.full((self.Tq, heads * dim + 16), -7.0, device="cuda", dtype=tdt)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.tables = [i32(self.cu), i32(self.begin), i32(kl)]
        self.scale = 1.0 / math.sqrt(dim)
        self.max_q, self.max_k = max(ql), max(kl)

    def args(self):
        kvd = self.kv_heads * self.dim
        return (self.q.data_ptr(), self.kv.data_ptr(), self.kv.data_ptr() + 2 * kvd, self.q.stride(0), 2 * kvd, 2 * kvd,
                *[t.data_ptr() for t in self.tables], len(self.ql), self.Tq, self.Tk, self.max_q, self.max_k, self.heads,
                self.kv_heads, self.dim, self.scale, DT[self.dtype], self.out.data_ptr(), self.out.stride(0))

    def run(self, stream=None):
        call(self.torch, *self.args(), stream=stream)
        return self.out

    def check(self, skip=()):
        torch, D, group = self.torch, self.dim, self.heads // self.kv_heads
        u = torch.finfo(self.out.dtype).eps / 2
        kvd = self.kv_heads * D
        worst = 0.0
        for s, (n, k) in enumerate(zip(self.ql, self.kl)):
            rows = slice(self.cu[s], self.cu[s] + n)
            if s in skip:
                assert bool((self.out[rows] == -7.0).all())
                continue
            keys = slice(self.begin[s], self.begin[s] + k)
            for h in range(self.heads):
                j = h // group * D
                q = self.q[rows, h * D:(h + 1) * D].double()
                K, V = self.kv[keys, j:j + D].double(), self.kv[keys, kvd + j:kvd + j + D].double()
                got = self.out[rows, h * D:(h + 1) * D].double()
                if k == 0:
                    assert bool((got == 0).all())
                    continue
                S = q @ K.t() * self.scale
                P = torch.softmax(S, 1)
                want, A = P @ V, P @ V.abs()
                mag = (q.abs() @ K.abs().t() * self.scale).amax(1, keepdim=True)
                d = D * 2.0**-23 * mag + (2.0**-22 + 2.0**-23) * (1 + 1.5 * S.abs().amax(1, keepdim=True))
                tol = u * (A + want.abs()) + 4 * d * A + 2.0**-17 * A + (k + 16) * 2.0**-23 * A + u * u * A
                if self.dtype == "f16":
                    tol = tol + 2.0**-25 * (V.abs().sum(0, keepdim=True) + 1)
                worst = max(worst, float(((got - want).abs() / tol).max())) if n else worst
        assert worst <= 1, worst
        assert bool((self.out[self.cu[-1]:] == -7.0).all()) and bool((self.out[:, self.heads * D:] == -7.0).all())


HEADS = [(2, 2, 32), (3, 3, 64), (4, 2, 128), (3, 1, 256)]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_one_token(cuda, heads, kv_heads, dim, dtype):
    """Single tokens over texts of one key, of the edges of a chunk, of none, and of several thousand."""
    kl = [1, 15, 16, 17, 0, 31, 33, 64, 127, 300, 0, 4000]
    b = Batch(cuda, [1] * len(kl), kl, heads, kv_heads, dim, dtype, 1 + dim)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("padded", [False, True])
def test_prompts(cuda, heads, kv_heads, dim, dtype, padded):
    """Prompts of one to several hundred tokens, at the edges of tiles and blocks; padded: NaN behind every text."""
    ql = [1, 127, 128, 129, 40, 0, 257, 300, 5, 200, 64]
    kl = [1, 63, 64, 65, 0, 70, 127, 128, 129, 500, 257]
    b = Batch(cuda, ql, kl, heads, kv_heads, dim, dtype, 2 + dim, padded=padded)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS + [(8, 1, 64), (16, 2, 128), (32, 1, 32)])
@pytest.mark.parametrize("q", [2, 5, 16])
def test_few_tokens(cuda, heads, kv_heads, dim, q):
    """A few tokens (rows of several heads share a tile), NaN behind the texts."""
    b = Batch(cuda, [q, 1, q, 0, q - 1], [100, 7, 1000, 50, 129], heads, kv_heads, dim, "bf16", q + dim, padded=True)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("ql,kl,heads,kv_heads,dim", [
    ([1], [9000], 1, 1, 128), ([1], [5000], 2, 1, 256), ([3], [20000], 4, 1, 64), ([1, 1], [12, 8000], 2, 2, 32),
    ([130], [6000], 1, 1, 128), ([300], [5000], 2, 1, 256), ([200], [4100], 2, 2, 64), ([500, 3], [8000, 40], 1, 1, 32),
])
def test_keys_split_over_a_cluster(cuda, ql, kl, heads, kv_heads, dim):
    """Little parallel work over long texts: the keys are split and the parts joined (one part may have no key)."""
    b = Batch(cuda, ql, kl, heads, kv_heads, dim, "bf16", sum(kl), padded=True)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("q", [1, 300])
@pytest.mark.parametrize("dim", [64, 256])
def test_no_text_has_a_key(cuda, q, dim):
    """Every text empty, max_kv 0: zeros, and rows outside the sequences left alone."""
    b = Batch(cuda, [q, 0, q], [0, 0, 0], 2, 1, dim, "f16", 31)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("ql,bound", [([1] * 3000, 1), ([1] * 400, 100), ([130] * 300, 130)])
def test_many_sequences(cuda, ql, bound):
    """Thousands of short sequences, and bounds far above the lengths (the kernel is chosen by the bounds)."""
    kl = [(13 * i) % 40 for i in range(len(ql))]
    b = Batch(cuda, ql, kl, 2, 2, 32, "bf16", 32)
    b.max_q, b.max_k = bound, 5000
    b.run()
    status(cuda)
    b.check()


def test_beside_a_projection_on_another_stream(cuda):
    """Calls that split their work over clusters, on two streams at once, leave each other's results alone."""
    import test_gpu_e4m3 as e4

    torch = cuda
    b = Batch(cuda, [130], [6000], 2, 2, 64, "bf16", 33)
    host, ops = e4.operands(torch, 37, 2048, 4096, 34)
    y = e4.dense(torch, ops, 37, 2048, 4096, None, "bf16")
    want, ref = b.run().clone(), y.clone()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        b.run(stream=s1.cuda_stream)
        e4.dense(torch, ops, 37, 2048, 4096, None, "bf16", stream=s2.cuda_stream, y=y)
    torch.cuda.synchronize()
    status(torch)
    assert torch.equal(b.out, want) and torch.equal(y, ref)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_many_items_of_a_few_blocks(cuda, heads, kv_heads, dim):
    """More (sequence, head, tile) items than SMs, most of one to three key blocks that end inside a 16-key step,
    with empty texts and empty prompts between."""
    kl = [(7 * i) % 90 + (130 if i % 5 == 0 else 0) if i % 9 else 0 for i in range(120)]
    ql = [(37 * i) % 300 if i % 11 else 0 for i in range(120)]
    b = Batch(cuda, ql, kl, heads, kv_heads, dim, "bf16", 13, padded=True)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("q", [1, 200])
def test_beams_share_a_text(cuda, q):
    b = Batch(cuda, [q] * 5, [333], 4, 2, 64, "bf16", 7, shared=True)
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("q", [1, 200])
def test_large_scores(cuda, q):
    """Scores in the hundreds: all the weight on one key, and a maximum that rises from block to block."""
    torch = cuda
    b = Batch(cuda, [q, q], [700, 256], 2, 1, 64, "bf16", 8)
    ramp = torch.linspace(0.1, 6.0, b.Tk, device="cuda")[:, None]
    b.kv[:, :64] = (b.kv[:, :64].float().abs() * ramp).to(b.kv.dtype)
    b.q[:, :128] = b.q[:, :128].abs()
    b.run()
    status(cuda)
    b.check()


@pytest.mark.parametrize("q", [1, 150])
def test_infinite_and_nan_values(cuda, q):
    """An infinity in one text's V and a NaN in another's K stay in their sequences."""
    torch = cuda
    b = Batch(cuda, [q, q, q], [40, 130, 64], 2, 2, 64, "bf16", 9)
    clean = b.run().clone()
    b.kv[40 + 129, 2 * 64 + 3] = float("inf")  # last key of the second text, V
    b.kv[40 + 130 + 5, 0] = float("nan")       # third text, K of head 0
    b.out.fill_(-7.0)
    dirty = b.run()
    status(torch)
    assert torch.equal(dirty[:q], clean[:q])
    second, third = slice(q, 2 * q), slice(2 * q, 3 * q)
    assert bool(torch.isinf(dirty[second, 3]).all())
    keep = [c for c in range(128) if c != 3]
    assert torch.equal(dirty[second][:, keep], clean[second][:, keep])
    assert bool(torch.isnan(dirty[third, :64]).all()) and torch.equal(dirty[third, 64:128], clean[third, 64:128])


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("q", [3, 150])
def test_infinite_scores(cuda, heads, kv_heads, dim, q):
    """An infinity in K at any place of a block: a query that meets it with a positive value is NaN (inf - inf), one
    with a negative value gives that key no weight."""
    torch = cuda
    for key in (0, 1, 5, 6, 7, 14, 15, 31, 40, 63, 64, 127, 130):
        b = Batch(cuda, [q], [140], heads, kv_heads, dim, "bf16", 40 + key)
        b.run()
        keep = [k for k in range(140) if k != key]
        without = Batch(cuda, [q], [139], heads, kv_heads, dim, "bf16", 1)
        without.q, without.kv = b.q, b.kv[keep].contiguous()
        without.out = torch.full_like(b.out, -7.0)
        without.Tq = b.Tq
        without.run()
        without.check()
        b.kv[key, 0] = float("inf")
        b.out.fill_(-7.0)
        got = b.run()[:q, :dim].double()
        status(torch)
        up = b.q[:q, 0] > 0
        assert bool(torch.isnan(got[up]).all())
        # the same weights from sums in another order: within what both may be off the exact result
        a, w = got[~up], without.out[:q, :dim].double()[~up]
        assert a.numel() == 0 or float((a - w).abs().max()) <= 4 * 2.0**-8 * float(b.kv[:, kv_heads * dim:].abs().float().max())


@pytest.mark.parametrize("q", [1, 150])
@pytest.mark.parametrize("table,value,who", [(2, 500, 1), (1, -1, 0), (1, 10**6, 1), (2, -5, 0), (0, -3, 0)])
def test_bad_tables_are_reported(cuda, q, table, value, who):
    """A length over its bound or rows outside the buffers: the sequence is skipped and the status says so."""
    from rembed_b200.embedder import RembedError

    b = Batch(cuda, [q, q], [100, 90], 2, 1, 64, "bf16", 10)
    b.tables[table][who] = value
    b.run()
    with pytest.raises(RembedError, match="shape"):
        status(cuda)
    b.check(skip=(who,))
    status(cuda)


@pytest.mark.parametrize("q,heads,kv_heads,dim", [(1, 4, 2, 128), (300, 4, 2, 128), (300, 3, 1, 256), (200, 2, 2, 64)])
def test_repeats_in_graphs_and_on_streams(cuda, q, heads, kv_heads, dim):
    """The same bits on every call: beside another call on another stream, and replayed with other lengths in the tables."""
    torch = cuda
    one = Batch(cuda, [q, q, 1], [700, 90, 5], heads, kv_heads, dim, "bf16", 11)
    two = Batch(cuda, [q, 2, q], [64, 700, 31], heads, kv_heads, dim, "bf16", 12)
    a, b = one.run().clone(), two.run().clone()
    torch.cuda.synchronize()
    one.out.fill_(-7.0), two.out.fill_(-7.0)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    one.run(stream=s1.cuda_stream)
    two.run(stream=s2.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(one.out, a) and torch.equal(two.out, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one.run()
    one.out.fill_(-7.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(one.out, a)
    one.kl = [70, 9, 0]
    one.tables[2].copy_(torch.tensor(one.kl, dtype=torch.int32))
    g.replay()
    status(torch)
    one.check()


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("q", [1, 260])
def test_bits_do_not_depend_on_memory_latency(cuda, heads, kv_heads, dim, q):
    """The same bits with cold caches, and while copies on another stream hold the loads up: no role of the kernel may
    run further ahead of another than its barriers can tell."""
    torch = cuda
    b = Batch(cuda, [q, q - 1, q, 5], [3000, 130, 1111, 64], heads, kv_heads, dim, "bf16", 21)
    want = b.run().clone()
    status(torch)
    junk = torch.empty((2, 1 << 27), device="cuda", dtype=torch.uint8)
    side = torch.cuda.Stream()
    for i in range(12):
        b.out.fill_(-7.0)
        junk[0].fill_(i)
        torch.cuda.synchronize()
        if i % 2:
            with torch.cuda.stream(side):
                for _ in range(4):
                    junk[1].copy_(junk[0])
        b.run()
        status(torch)
        assert torch.equal(b.out, want)
    torch.cuda.synchronize()


def test_states_to_keys_to_attention(cuda):
    """The operators one after another, as they are used: an encoder's packed float32 states are quantised, projected
    to K and V in 8 bits, and attended to by a prompt, then by single tokens.  The attention is held to its own inputs;
    K and V to the exact projection within the operands' rounding."""
    from rembed_b200.embedder import library

    torch = cuda
    lens, H, heads, dim = [40, 7, 131], 768, 4, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    states = torch.randn((sum(lens), H), device="cuda", generator=g)
    w = torch.randn((2 * heads * dim, H), device="cuda", generator=g) * 0.03
    T, N = states.shape[0], w.shape[0]
    u8 = lambda r: torch.empty((r, H), device="cuda", dtype=torch.uint8)  # noqa: E731
    xq, wq, xs, ws = u8(T), u8(N), torch.empty((6, T), device="cuda"), torch.empty((4, 6), device="cuda")
    lib, st, err = library(), torch.cuda.current_stream().cuda_stream, ctypes.c_char_p()
    b = Batch(cuda, [60, 1, 9], lens, heads, heads, dim, "bf16", 4)
    assert lib.rg_quantize_tiles_e4m3(w.data_ptr(), 0, H, N, H, wq.data_ptr(), H, ws.data_ptr(), st, ctypes.byref(err)) == 0
    assert lib.rg_quantize_rows_e4m3(states.data_ptr(), 0, H, T, H, xq.data_ptr(), H, xs.data_ptr(), T, st, ctypes.byref(err)) == 0
    assert lib.rg_dense_e4m3(xq.data_ptr(), H, xs.data_ptr(), T, wq.data_ptr(), H, ws.data_ptr(), None, b.kv.data_ptr(), N, 2, T, N, H,
                             st, ctypes.byref(err)) == 0
    b.run()
    for _ in range(3):  # decoder steps over the same K and V
        step = Batch(cuda, [1, 1, 1], lens, heads, heads, dim, "bf16", 5)
        step.kv = b.kv
        step.run()
        step.check()
    status(torch)
    b.check()
    exact = states.double() @ w.double().t()
    rel = float((b.kv.double() - exact).norm() / exact.norm())
    assert rel <= math.sqrt(2) * 2.0**-3 / math.sqrt(12) + 2.0**-8


FIRST_IN_GRAPH = """
import ctypes, sys
sys.path[:0] = {paths!r}
import torch
import test_gpu_cross_attention as t
from rembed_b200.embedder import library
err = ctypes.c_char_p()
assert library().rg_kernel_status(None, ctypes.byref(err)) == 0
calls = [t.Batch(torch, q, [700, 2000], heads, kv_heads, dim, "bf16", 5)
         for q, heads, kv_heads, dim in (([1, 1], 4, 2, 64), ([300, 200], 4, 2, 128), ([150, 3], 3, 1, 256))]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    for c in calls:
        c.run()
g.replay()
t.status(torch)
for c in calls:
    c.check()
"""


def test_first_calls_in_a_capture(cuda):
    """Once the device has its status word, a kernel's first call may be one that is captured."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST_IN_GRAPH.format(paths=[os.path.dirname(here), here])], timeout=300,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("nseq,q,keys,heads,kv_heads,dim", [
    (2, 40, 4096, 3, 1, 256), (2, 128, 4096, 3, 1, 256), (1, 96, 4096, 3, 1, 256), (2, 200, 4096, 8, 1, 128),
    (1, 200, 4096, 16, 8, 128), (4, 64, 4096, 12, 12, 64), (1, 64, 2048, 12, 12, 64), (2, 64, 4096, 12, 12, 32),
])
def test_few_long_texts(cuda, nseq, q, keys, heads, kv_heads, dim):
    """Keys split over clusters of every size, as the SMs have room for them, by the rows' kernel and by the tiles'."""
    one = Batch(cuda, [q - s for s in range(nseq)], [keys - 100 * s for s in range(nseq)], heads, kv_heads, dim, "bf16", 21)
    one.run()
    status(cuda)
    one.check()
