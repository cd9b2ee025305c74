"""rg_cross_attention at the ends of its range: scores far beyond what a probability's exponent holds, rows
whose every score is -infinity, the many small probabilities of a long text, and buffers of gigabytes.  Then the
operators behind an encoder's forward pass."""

import ctypes
import math

import numpy as np
import pytest

from test_gpu_cross_attention import HEADS, Batch, status

pytestmark = pytest.mark.gpu

INF = float("inf")


def exact_rows(torch, b, scale):
    """The float64 result of every row of b's first sequence, and the bound on what the kernels may be off it, for
    scores that are exact in fp32.  With u half a step of the type and A = sum_j p_j |v_j|: probabilities and result
    are rounded (u A and u |o|, and their product); weights above 2^-30 have exponents of at most 30, so that scale's
    and the product's roundings (2^-24 of them each), the hardware exponential (2^-22) and the polynomial (2^-18)
    move them by at most 2^-16 in all, and where scores pass 2^10 in the exponent its rounding there by 2^-14; the
    sums' additions add (keys + 16) 2^-23 A, and in fp16 small probabilities keep 2^-25 absolute."""
    D, group, n, k = b.dim, b.heads // b.kv_heads, b.ql[0], b.kl[0]
    u = torch.finfo(b.out.dtype).eps / 2
    want, tol = [], []
    for h in range(b.heads):
        j = h // group * D
        K, V = b.kv[:k, j:j + D].double(), b.kv[:k, b.kv_heads * D + j:b.kv_heads * D + j + D].double()
        S = b.q[:n, h * D:(h + 1) * D].double() @ K.t() * scale
        P = torch.softmax(S, 1)
        o, A = P @ V, P @ V.abs()
        want.append(o)
        tol.append(u * (A + o.abs()) + u * u * A + (2.0**-16 + 2.0**-14) * A + (k + 16) * 2.0**-23 * A + 2.0**-25 * V.abs().sum(0))
    return torch.cat(want, 1), torch.cat(tol, 1)


def check_exact(torch, b):
    b.run()
    status(torch)
    want, tol = exact_rows(torch, b, b.scale)
    got = b.out[:b.ql[0], :b.heads * b.dim].double()
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).nan_to_num(INF).max())


def signs(torch, n):
    return torch.where(torch.arange(n, device="cuda") % 3 == 1, -1.0, 1.0)[:, None]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q", [1, 5, 150])
def test_scores_of_hundreds_of_millions(cuda, heads, kv_heads, dim, dtype, q):
    """Finite queries and keys of several thousand: scores up to 10^9, whose products with the scale are rounded to
    steps of 64 and more.  All the weight lies on the largest score, shared by equal ones.  Every score is exact in
    fp32: 32 equal products of an 8- or 10-bit and a 7-bit number."""
    torch = cuda
    b = Batch(torch, [q], [700], heads, kv_heads, dim, dtype, 70 + dim)
    g = torch.Generator(device="cuda").manual_seed(dim)
    r = torch.randint(1, 128, (700, kv_heads), device="cuda", generator=g).float()
    b.q.zero_()
    b.kv[:, :kv_heads * dim] = 0
    for h in range(heads):
        b.q[:q, h * dim:h * dim + 32] = (signs(torch, q) * (6976.0 if dtype == "bf16" else 7000.0)).to(b.q.dtype)
    for h in range(kv_heads):
        b.kv[:, h * dim:h * dim + 32] = (64 * r[:, h:h + 1]).to(b.kv.dtype)
    b.scale = 0.37
    check_exact(torch, b)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q", [1, 5, 150])
@pytest.mark.parametrize("base", [2.0**11, -2.0**11, 2.0**8])
def test_small_differences_of_large_scores(cuda, heads, kv_heads, dim, dtype, q, base):
    """Scores of several millions (of a million: base 2^8) that differ by small whole numbers, exact in fp32, and a
    text that begins with keys of small scores: those of larger ones take all the weight, by their differences."""
    torch = cuda
    b = Batch(torch, [q], [700], heads, kv_heads, dim, dtype, 80 + dim)
    g = torch.Generator(device="cuda").manual_seed(dim)
    b.q.zero_()
    b.kv[:, :kv_heads * dim] = 0
    for h in range(heads):
        b.q[:q, h * dim] = 4096.0
        b.q[:q, h * dim + 1] = 1.0
    for h in range(kv_heads):
        b.kv[130:, h * dim] = base
        b.kv[:, h * dim + 1] = torch.randint(0, 16, (700,), device="cuda", generator=g).to(b.kv.dtype)
    b.scale = 0.37
    check_exact(torch, b)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q", [2, 5, 150])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_pass_a_thousand(cuda, heads, kv_heads, dim, dtype, q, falling):
    """Maxima that rise or fall through 2^10 and -2^10 in the exponent, by steps of 8.5 with differences within them."""
    torch = cuda
    b = Batch(torch, [q], [700], heads, kv_heads, dim, dtype, 85 + dim)
    g = torch.Generator(device="cuda").manual_seed(dim)
    b.q.zero_()
    b.kv[:, :kv_heads * dim] = 0
    ramp = torch.div(torch.arange(700, device="cuda") * 16, 700, rounding_mode="floor") + 112
    for h in range(heads):
        b.q[:q, h * dim] = 16 * signs(torch, q)[:, 0].to(b.q.dtype)
        b.q[:q, h * dim + 1] = 1.0
    for h in range(kv_heads):
        b.kv[:, h * dim] = (ramp.flip(0) if falling else ramp).to(b.kv.dtype)
        b.kv[:, h * dim + 1] = torch.randint(0, 16, (700,), device="cuda", generator=g).to(b.kv.dtype)
    b.scale = 0.37
    check_exact(torch, b)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("q", [1, 5, 150])
@pytest.mark.parametrize("dtype,query,step,scale", [
    ("bf16", 1.5 * 2.0**60, 2.0**53, 1000.0), ("bf16", 1.0, 1.0, 2.0e38), ("f16", 1.0, 1.0, 2.0e38),
])
def test_scores_that_overflow_with_the_scale(cuda, heads, kv_heads, dim, q, dtype, query, step, scale):
    """Finite scores whose product with an allowed scale is none in fp32: the largest takes all the weight."""
    torch = cuda
    b = Batch(torch, [q], [300], heads, kv_heads, dim, dtype, 90 + dim)
    g = torch.Generator(device="cuda").manual_seed(dim)
    b.q.zero_()
    b.kv[:, :kv_heads * dim] = 0
    for h in range(heads):
        b.q[:q, h * dim] = (signs(torch, q)[:, 0] * query).to(b.q.dtype)
    for h in range(kv_heads):
        b.kv[:, h * dim] = (step * torch.randint(2, 128, (300,), device="cuda", generator=g).float()).to(b.kv.dtype)
    b.scale = scale
    check_exact(torch, b)


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q", [3, 150])
def test_rows_of_minus_infinities(cuda, heads, kv_heads, dim, dtype, q):
    """Keys that hold an infinity, met by negative queries.  Where a text has no other key the softmax is 0 / 0: NaN, of
    one key as of many, and for every place in a block.  Where it has others, the result is theirs."""
    torch = cuda
    kl = [1, 3, 140, 300, 50]
    hidden = [range(1), range(3), range(140), range(260), range(0)]  # the keys with an infinity
    b = Batch(torch, [q] * len(kl), kl, heads, kv_heads, dim, dtype, 50 + dim)
    b.q[:, :heads * dim:dim] = -b.q[:, :heads * dim:dim].abs() - 0.5
    clean = b.run().clone()
    for at, keys in zip(b.begin, hidden):
        if len(keys):
            b.kv[at + keys[0]:at + keys[-1] + 1, :kv_heads * dim:dim] = INF
    b.out.fill_(-7.0)
    got = b.run()[:, :heads * dim]
    status(torch)
    assert bool(torch.isnan(got[:3 * q]).all())
    assert torch.equal(got[4 * q:5 * q], clean[4 * q:5 * q, :heads * dim])
    rest = Batch(torch, [0, 0, 0, q, 0], kl, heads, kv_heads, dim, dtype, 1)
    rest.q, rest.kv, rest.Tq = b.q[3 * q:].contiguous(), b.kv, q + 3
    rest.begin[3] += 260
    rest.kl[3] -= 260
    rest.tables[1][3] += 260
    rest.tables[2][3] -= 260
    rest.out = torch.full((q + 3, heads * dim + 16), -7.0, device="cuda", dtype=b.out.dtype)
    rest.run()
    status(torch)
    rest.check()
    # the same weights from sums in another order: within what both may be off the exact result
    v = b.kv[b.begin[3]:b.begin[3] + 300, kv_heads * dim:].float().abs().max()
    u = torch.finfo(b.out.dtype).eps / 2
    assert float((got[3 * q:4 * q].float() - rest.out[:q, :heads * dim].float()).abs().max()) <= 4 * u * float(v)


@pytest.mark.parametrize("q,keys,heads,kv_heads,dim", [
    (1, 9000, 1, 1, 128), (1, 5000, 2, 1, 256), (3, 20000, 4, 1, 64), (130, 6000, 1, 1, 128), (300, 5000, 2, 1, 256),
    (200, 4100, 2, 2, 64), (500, 8000, 1, 1, 32),
])
def test_minus_infinities_in_split_keys(cuda, q, keys, heads, kv_heads, dim):
    """The same where the keys are split over a cluster: all parts without weight (NaN), then all but the last key's."""
    torch = cuda
    b = Batch(torch, [q], [keys], heads, kv_heads, dim, "bf16", 60 + dim)
    b.q[:, :heads * dim:dim] = -b.q[:, :heads * dim:dim].abs() - 0.5
    b.kv[:, :kv_heads * dim:dim] = INF
    assert bool(torch.isnan(b.run()[:q, :heads * dim]).all())
    b.kv[keys - 1, :kv_heads * dim:dim] = 1.0
    got = b.run()[:q, :heads * dim]
    status(torch)
    v = b.kv[keys - 1, kv_heads * dim:].view(kv_heads, 1, dim).expand(kv_heads, heads // kv_heads, dim).reshape(1, -1)
    assert torch.equal(got, v.expand(q, -1))


@pytest.mark.parametrize("q,heads,kv_heads,dim", [(1, 1, 1, 32), (3, 2, 2, 64), (2000, 1, 1, 64), (2000, 2, 1, 128), (1500, 1, 1, 256)])
def test_many_small_probabilities_in_fp16(cuda, q, heads, kv_heads, dim):
    """One key with nearly all the weight over a text of 2^17: the others' 2^-27 each are below the steps of fp16, but
    a thousandth together.  V is 0 at the first and 1 at the others, so that the result is that thousandth, off by its
    rounding (2^-11), the probabilities' (2^-11, or 2^-25 of the largest value of P there is, 2^7 and more), the
    exponentials' (2^-16) and the sums' additions ((keys + 16) 2^-23 of it)."""
    torch = cuda
    n = 1 << 17
    b = Batch(torch, [q], [n], heads, kv_heads, dim, "f16", 99)
    b.q.zero_()
    b.kv.zero_()
    b.q[:q, :heads * dim:dim] = 1.0
    b.kv[0, :kv_heads * dim:dim] = 18.75
    b.kv[1:, kv_heads * dim:] = 1.0
    b.scale = 1.0
    b.run()
    status(torch)
    w = (n - 1) * math.exp(-18.75)
    want = w / (1 + w)
    got = b.out[:q, :heads * dim].double()
    assert float((got - want).abs().max()) <= (2.0**-10 + 2.0**-16 + (n + 16) * 2.0**-23) * want + n * 2.0**-32


@pytest.mark.parametrize("q", [1, 3, 200])
@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 4, 128), (16, 2, 256)])
def test_texts_and_rows_beyond_2_32_bytes(cuda, q, heads, kv_heads, dim):
    """A text at the end of a cache of 8 GiB, queries and outputs at the end of buffers of 8 GiB, with anything before."""
    torch = cuda
    b = Batch(torch, [q, q], [700, 41], heads, kv_heads, dim, "bf16", 95)
    first_q, first_k = 2**20, 2**22
    big = lambda rows, like: torch.empty((rows + like.shape[0], like.shape[1]), device="cuda", dtype=like.dtype)  # noqa: E731
    far = Batch(torch, [q, q], [700, 41], heads, kv_heads, dim, "bf16", 95)
    far.q, far.kv, far.out = big(first_q, b.q), big(first_k, b.kv), big(first_q, b.out)
    far.q[first_q:], far.kv[first_k:], far.out[first_q:] = b.q, b.kv, -7.0
    assert far.q.numel() > 2**32 and far.kv.numel() >= 2**32 and far.out.numel() > 2**32
    far.tables[0] += first_q
    far.tables[1] += first_k
    far.Tq += first_q
    far.Tk += first_k
    b.run()
    far.run()
    status(torch)
    b.check()
    assert torch.equal(far.out[first_q:], b.out)


def test_behind_an_encoder(cuda):
    """An encoder's forward pass leaves its token states on the device; they are quantised, projected to K and V, and
    attended to by prompts and then by single tokens, all on one stream without a synchronisation.  K and V are held to
    the exact projection of the states (within the operands' 8-bit rounding), the attention to its inputs."""
    from rembed_b200 import synth
    from rembed_b200.embedder import Embedder, library

    torch = cuda
    lens, heads, dim = [40, 7, 131], 4, 64
    cfg = synth.preset("minilm-l6")
    enc = Embedder(cfg, synth.make_weights(cfg, seed=0))
    H, T, N = cfg.hidden_size, sum(lens), 2 * heads * dim
    cu = np.cumsum([0] + lens).astype(np.int32)
    rng = np.random.default_rng(3)
    ids = rng.integers(1000, 30000, T)
    d_ids, d_cu = torch.from_numpy(ids).cuda(), torch.from_numpy(cu).cuda()
    w = torch.randn((N, H), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)) * 0.03
    states = torch.empty((T, H), device="cuda")
    xq, wq = (torch.empty((r, H), device="cuda", dtype=torch.uint8) for r in (T, N))
    xs, ws = torch.empty((H // 128, T), device="cuda"), torch.empty((N // 128, H // 128), device="cuda")
    prompt = Batch(torch, [60, 1, 9], lens, heads, heads, dim, "bf16", 4)
    step = Batch(torch, [1, 1, 1], lens, heads, heads, dim, "bf16", 5)
    step.kv = prompt.kv
    torch.cuda.synchronize()
    lib, err, at = library(), ctypes.c_char_p(), torch.cuda.Stream().cuda_stream
    enc.forward_device(d_ids.data_ptr(), d_cu.data_ptr(), cu, states.data_ptr(), stream=at, tokens=True)
    assert lib.rg_quantize_tiles_e4m3(w.data_ptr(), 0, H, N, H, wq.data_ptr(), H, ws.data_ptr(), at, ctypes.byref(err)) == 0
    assert lib.rg_quantize_rows_e4m3(states.data_ptr(), 0, H, T, H, xq.data_ptr(), H, xs.data_ptr(), T, at, ctypes.byref(err)) == 0
    assert lib.rg_dense_e4m3(xq.data_ptr(), H, xs.data_ptr(), T, wq.data_ptr(), H, ws.data_ptr(), None, prompt.kv.data_ptr(), N, 2,
                             T, N, H, at, ctypes.byref(err)) == 0
    prompt.run(stream=at)
    step.run(stream=at)
    torch.cuda.synchronize()
    enc.sync()
    status(torch)
    vectors = enc.embed_tokens([ids[a:b] for a, b in zip(cu[:-1], cu[1:])])
    assert np.array_equal(states.cpu().numpy(), np.concatenate([v.vectors for v in vectors]))
    exact = states.double() @ w.double().t()
    # independent errors of two factors, each of rms below 2^-3 / sqrt(12) of itself, and the result's rounding
    assert float((prompt.kv.double() - exact).norm() / exact.norm()) <= math.sqrt(2) * 2.0**-3 / math.sqrt(12) + 2.0**-8
    prompt.check()
    step.check()
