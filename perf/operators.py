"""Cases of the 8-bit block-scaled projection and of cross attention, for timing and comparison.

Three operators, as a decoder over this library's encoder states uses them: the states are quantised to
e4m3 with a float32 scale for each block of 128 (`rg_quantize_rows_e4m3`, the weights once by
`rg_quantize_tiles_e4m3`), projected by `rg_dense_e4m3`, and attended to by `rg_cross_attention`.

`run` computes them in elementary torch operations in float32 where `own` is false, and through the
library's entry points where it is true.
"""

import ctypes
import math
import random

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
RG_DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def _up(a, b):
    return -(-a // b) * b


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one step of a decoder: eight running texts' activations before a projection
        dict(name="quantize_rows_step", op="rows", M=8, K=1024, dtype="bf16"),
        # the encoder's float32 token states of a packed batch (widest hidden size served: 1024), an odd number of tokens
        dict(name="quantize_rows_states", op="rows", M=98305, K=1024, dtype="f32"),
        # a ragged width: 1100 columns end inside a block
        dict(name="quantize_rows_ragged", op="rows", M=4099, K=1100, dtype="f16"),
        # a weight, quantised once at load: 128 x 128 tiles
        dict(name="quantize_tiles_weight", op="tiles", N=4096, K=4096, dtype="f32"),
        # one token through a Q projection of 16 heads x 128
        dict(name="dense_one_token", op="dense", M=1, N=2048, K=1024, dtype="bf16", bias=False),
        # a serving batch of single tokens through a wide feed-forward weight: the weight's bytes count
        dict(name="dense_few_rows", op="dense", M=37, N=8192, K=4096, dtype="bf16", bias=False),
        # K and V of a few texts' states, fused and with a bias, sizes that divide by nothing
        dict(name="dense_odd", op="dense", M=1003, N=1540, K=1100, dtype="f16", bias=True),
        # K and V of a large packed batch of states
        dict(name="dense_large", op="dense", M=16384, N=4096, K=4096, dtype="bf16", bias=True),
        # one decoder token for each of 64 texts, the states of BERT-base-like heads, texts of 1 to 512 tokens
        dict(name="cross_one_token", op="cross", B=64, q_lo=1, q_hi=1, k_lo=1, k_hi=512, heads=12, kv_heads=12, dim=64, dtype="bf16", empty=0, padded=False),
        # one decoder token for each of 4 long documents, grouped heads: K and V are read once, nothing else counts
        dict(name="cross_one_token_long", op="cross", B=4, q_lo=1, q_hi=1, k_lo=24000, k_hi=32768, heads=16, kv_heads=8, dim=128, dtype="f16", empty=0, padded=False),
        # ragged prompts over ragged texts in a padded buffer, some of the texts empty
        dict(name="cross_prompts_ragged", op="cross", B=24, q_lo=1, q_hi=300, k_lo=1, k_hi=700, heads=3, kv_heads=1, dim=256, dtype="bf16", empty=3, padded=True),
        # long targets over long documents: the largest
        dict(name="cross_prompts_long", op="cross", B=8, q_lo=1500, q_hi=2048, k_lo=3000, k_hi=4096, heads=16, kv_heads=8, dim=128, dtype="bf16", empty=0, padded=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi))))


def _cross_cost(c):
    return c["B"] * c["heads"] * c["q_hi"] * c["k_hi"] * c["dim"], c["B"] * c["k_hi"] * c["kv_heads"] * c["dim"]


def draw(rng):
    op = rng.choice(["rows", "tiles", "dense", "dense", "cross", "cross"])
    while True:
        if op == "rows":
            c = dict(op=op, M=_log(rng, 1, 100000), K=_log(rng, 1, 8192), dtype=rng.choice(list(DTYPES)))
            if c["M"] * c["K"] <= 98305 * 1024:
                return c
        elif op == "tiles":
            c = dict(op=op, N=_log(rng, 1, 16384), K=_log(rng, 1, 16384), dtype=rng.choice(list(DTYPES)))
            if c["N"] * c["K"] <= 4096 * 4096:
                return c
        elif op == "dense":
            c = dict(op=op, M=_log(rng, 1, 32768), N=_log(rng, 16, 8192), K=_log(rng, 32, 8192), dtype=rng.choice(list(DTYPES)), bias=rng.random() < 0.5)
            if c["M"] * c["N"] * c["K"] <= 16384 * 4096 * 4096:
                return c
        else:
            heads, kv_heads, dim = rng.choice([(12, 12, 32), (12, 12, 64), (16, 8, 128), (3, 1, 256), (8, 1, 128), (6, 3, 64)])
            q_hi = 1 if rng.random() < 0.4 else _log(rng, 2, 2048)
            k_hi = _log(rng, 1, 32768)
            B = _log(rng, 1, 64)
            c = dict(op=op, B=B, q_lo=max(1, q_hi // rng.randint(1, 8)), q_hi=q_hi, k_lo=max(1, k_hi // rng.randint(1, 8)), k_hi=k_hi, heads=heads, kv_heads=kv_heads,
                     dim=dim, dtype=rng.choice(["f16", "bf16"]), empty=rng.randint(0, B // 4), padded=rng.random() < 0.5)
            if _cross_cost(c)[0] <= 8 * 16 * 2048 * 4096 * 128 and _cross_cost(c)[1] <= 4 * 32768 * 8 * 128:
                return c


def _lengths(c):
    """Query and key lengths of a cross case: they belong to the case, so that its work is known."""
    r = random.Random("%(B)d %(q_lo)d %(q_hi)d %(k_lo)d %(k_hi)d %(empty)d" % c)
    ql = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["B"])]
    kl = [r.randint(c["k_lo"], c["k_hi"]) for _ in range(c["B"])]
    for i in r.sample(range(c["B"]), c["empty"]):
        kl[i] = 0
    return ql, kl


def work(case):
    c = case
    if c["op"] in ("rows", "tiles"):
        n = (c["M"] if c["op"] == "rows" else c["N"]) * c["K"]
        kb = -(-c["K"] // BLOCK)
        scales = c["M"] * kb if c["op"] == "rows" else -(-c["N"] // BLOCK) * kb
        return {"bytes": n * (SIZES[c["dtype"]] + 1) + 4 * scales, "flops": 2 * n}
    if c["op"] == "dense":
        M, N, K = c["M"], c["N"], c["K"]
        kb = -(-K // BLOCK)
        return {"bytes": M * K + N * K + 4 * kb * (M + -(-N // BLOCK)) + (4 * N if c["bias"] else 0) + M * N * SIZES[c["dtype"]], "flops": 2 * M * N * K}
    ql, kl = _lengths(c)
    size = SIZES[c["dtype"]]
    return {"bytes": size * c["dim"] * (2 * sum(ql) * c["heads"] + 2 * sum(kl) * c["kv_heads"]) + 4 * (3 * c["B"] + 1),
            "flops": 4 * c["heads"] * c["dim"] * sum(a * b for a, b in zip(ql, kl))}


# ---------------------------------------------------------------- inputs

def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _states(g, rows, cols):
    """Token states as an encoder's last norm leaves them: unit variance, a few channels far louder."""
    x = _normal(g, rows, cols)
    return x * torch.exp(0.5 * _normal(g, cols)).add_(8.0 * (torch.rand(cols, device="cuda", generator=g) < 0.01))


def _rows_e4m3(x):
    """Elementary form: x [M x K] -> e4m3 [M x K] and the scales [K blocks x M]."""
    M, K = x.shape
    kb = -(-K // BLOCK)
    f = torch.zeros((M, kb * BLOCK), device=x.device)
    f[:, :K] = x
    f = f.view(M, kb, BLOCK)
    amax = f.abs().amax(2)
    scale = torch.where(amax == 0, torch.ones_like(amax), torch.clamp(amax / E4M3_MAX, min=2.0**-126))
    q = (f * (1.0 / scale)[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(M, kb * BLOCK)[:, :K].contiguous(), scale.t().contiguous()


def _tiles_e4m3(w):
    """Elementary form: w [N x K] -> e4m3 [N x K] and the scales [N blocks x K blocks]."""
    N, K = w.shape
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    f = torch.zeros((nb * BLOCK, kb * BLOCK), device=w.device)
    f[:N, :K] = w
    f = f.view(nb, BLOCK, kb, BLOCK)
    amax = f.abs().amax((1, 3))
    scale = torch.where(amax == 0, torch.ones_like(amax), torch.clamp(amax / E4M3_MAX, min=2.0**-126))
    q = (f * (1.0 / scale)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(nb * BLOCK, kb * BLOCK)[:N, :K].contiguous(), scale


def _aligned(q):
    """e4m3 rows at a stride that is a multiple of 16 bytes, as the projection reads them."""
    buf = torch.zeros((q.shape[0], _up(q.shape[1], 16)), device=q.device, dtype=torch.uint8)
    buf[:, : q.shape[1]] = q.view(torch.uint8)
    return buf


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["op"] == "rows":
        return dict(c, x=_states(g, c["M"], c["K"]).to(DTYPES[c["dtype"]]))
    if c["op"] == "tiles":
        return dict(c, x=(0.02 * _normal(g, c["N"], c["K"])).to(DTYPES[c["dtype"]]))
    if c["op"] == "dense":
        xq, xs = _rows_e4m3(_states(g, c["M"], c["K"]))
        wq, ws = _tiles_e4m3(0.02 * _normal(g, c["N"], c["K"]))
        return dict(c, xq=_aligned(xq), xs=xs, wq=_aligned(wq), ws=ws, b=0.02 * _normal(g, c["N"]) if c["bias"] else None)
    # cross attention: queries a little wider than keys, so that the softmax has favourites
    ql, kl = _lengths(c)
    dt = DTYPES[c["dtype"]]
    at = [i * c["k_hi"] for i in range(c["B"])] if c["padded"] else [sum(kl[:i]) for i in range(c["B"])]
    Tq, Tk = sum(ql), max(1, c["B"] * c["k_hi"] if c["padded"] else sum(kl))
    kvd = c["kv_heads"] * c["dim"]
    q = (1.5 * _normal(g, Tq, c["heads"] * c["dim"])).to(dt)
    kv = _normal(g, Tk, 2 * kvd).to(dt)  # K and V as one projection of the states leaves them
    cu = torch.tensor([sum(ql[:i]) for i in range(c["B"] + 1)], dtype=torch.int32, device="cuda")
    return dict(c, q=q, kv=kv, cu=cu, begin=torch.tensor(at, dtype=torch.int32, device="cuda"), length=torch.tensor(kl, dtype=torch.int32, device="cuda"),
                max_q=max(ql), max_k=max(max(kl), 1))


# ---------------------------------------------------------------- the plain forms

def _dense_plain(s):
    K, N = s["K"], s["N"]
    x = s["xq"][:, :K].view(torch.float8_e4m3fn).float() * s["xs"].t().repeat_interleave(BLOCK, 1)[:, :K]
    w = s["wq"][:, :K].view(torch.float8_e4m3fn).float() * s["ws"].repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    y = x @ w.t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["dtype"]])


def _cross_plain(s):
    H, G, D, B = s["heads"], s["kv_heads"], s["dim"], s["B"]
    q, kv = s["q"], s["kv"]
    qi, ki = torch.arange(s["max_q"], device="cuda"), torch.arange(s["max_k"], device="cuda")
    start, qlen = s["cu"][:-1, None], (s["cu"][1:] - s["cu"][:-1])[:, None]
    rows = torch.clamp(start + qi, max=q.shape[0] - 1)  # [B, max_q], past a sequence's end: any row
    keys = torch.clamp(s["begin"][:, None] + ki, max=kv.shape[0] - 1)
    valid = ki < s["length"][:, None]  # [B, max_k]
    Q = q[rows.long()].float().view(B, s["max_q"], G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    KV = kv[keys.long()].float().view(B, s["max_k"], 2, G, D)
    KV = torch.where(valid[:, :, None, None, None], KV, torch.zeros_like(KV))
    Kt, V = KV[:, :, 0].permute(0, 2, 3, 1), KV[:, :, 1].permute(0, 2, 1, 3)
    S = Q @ Kt
    S *= 1.0 / math.sqrt(D)
    S.masked_fill_(~valid[:, None, None, :], -math.inf)
    S -= S.amax(3, keepdim=True).clamp(min=-1e30)
    P = S.exp_()
    O = (P @ V) / P.sum(3, keepdim=True).clamp(min=1e-30)  # no key: zeros
    O = O.view(B, G, H // G, s["max_q"], D).permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], H * D)
    out = torch.empty_like(q)
    at = torch.where(qi < qlen, rows, q.shape[0])  # rows past a sequence's end go to a row of their own
    full = torch.cat([out, out[:1]])
    full[at.long().view(-1)] = O.view(-1, H * D).to(q.dtype)
    return full[:-1]


# ---------------------------------------------------------------- the library's calls

def _call(name, *args):
    from rembed_b200.embedder import RembedError, library, take_error

    err = ctypes.c_char_p()
    if getattr(library(), name)(*args, torch.cuda.current_stream().cuda_stream, ctypes.byref(err)) != 0:
        raise RembedError(take_error(err))


def _own(s):
    if s["op"] in ("rows", "tiles"):
        x = s["x"]
        rows, K = x.shape
        kb = -(-K // BLOCK)
        q = torch.empty((rows, _up(K, 16)), device="cuda", dtype=torch.uint8)
        if s["op"] == "rows":
            scale = torch.empty((kb, rows), device="cuda")
            _call("rg_quantize_rows_e4m3", x.data_ptr(), RG_DTYPES[s["dtype"]], K, rows, K, q.data_ptr(), q.stride(0), scale.data_ptr(), rows)
        else:
            scale = torch.empty((-(-rows // BLOCK), kb), device="cuda")
            _call("rg_quantize_tiles_e4m3", x.data_ptr(), RG_DTYPES[s["dtype"]], K, rows, K, q.data_ptr(), q.stride(0), scale.data_ptr())
        return q[:, :K].view(torch.float8_e4m3fn), scale
    if s["op"] == "dense":
        y = torch.empty((s["M"], s["N"]), device="cuda", dtype=DTYPES[s["dtype"]])
        _call("rg_dense_e4m3", s["xq"].data_ptr(), s["xq"].stride(0), s["xs"].data_ptr(), s["M"], s["wq"].data_ptr(), s["wq"].stride(0), s["ws"].data_ptr(),
              None if s["b"] is None else s["b"].data_ptr(), y.data_ptr(), s["N"], RG_DTYPES[s["dtype"]], s["M"], s["N"], s["K"])
        return y
    q, kv, kvd = s["q"], s["kv"], s["kv_heads"] * s["dim"]
    out = torch.empty_like(q)
    _call("rg_cross_attention", q.data_ptr(), kv.data_ptr(), kv.data_ptr() + 2 * kvd, q.stride(0), kv.stride(0), kv.stride(0), s["cu"].data_ptr(), s["begin"].data_ptr(),
          s["length"].data_ptr(), s["B"], q.shape[0], kv.shape[0], s["max_q"], s["max_k"], s["heads"], s["kv_heads"], s["dim"], 1.0 / math.sqrt(s["dim"]),
          RG_DTYPES[s["dtype"]], out.data_ptr(), out.stride(0))
    return out


def run(state):
    if own:
        return _own(state)
    if state["op"] == "rows":
        return _rows_e4m3(state["x"])
    if state["op"] == "tiles":
        return _tiles_e4m3(state["x"])
    return _dense_plain(state) if state["op"] == "dense" else _cross_plain(state)


# ---------------------------------------------------------------- the definitions in 64 bits

def _nearest_e4m3(x):
    """The e4m3 value next to x (ties to the even one): steps of 2^(e - 3), e the exponent of x and at least -6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), torch.clamp(e - 1, min=-6) - 3)
    return torch.clamp(torch.round(x / step) * step, -E4M3_MAX, E4M3_MAX)


def _exact_quantize(x, tiles):
    q = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    rows, K = x.shape
    tall = BLOCK if tiles else rows
    scales = []
    for r in range(0, rows, tall):
        for k in range(0, K, BLOCK):
            b = x[r : r + tall, k : k + BLOCK].double()
            s = (b.abs().max() if tiles else b.abs().amax(1)) / E4M3_MAX
            s = torch.where(s == 0, torch.ones_like(s), s)
            q[r : r + tall, k : k + BLOCK] = _nearest_e4m3(b / (s if tiles else s[:, None]))
            scales.append(s)
    scale = torch.stack(scales)
    return q, scale.view(-(-rows // BLOCK), -1) if tiles else scale


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("rows", "tiles"):
        return _exact_quantize(s["x"], c["op"] == "tiles")
    if c["op"] == "dense":
        y = torch.zeros((c["M"], c["N"]), dtype=torch.float64, device="cuda")
        for k in range(0, c["K"], BLOCK):
            e = min(k + BLOCK, c["K"])
            part = s["xq"][:, k:e].view(torch.float8_e4m3fn).double() @ s["wq"][:, k:e].view(torch.float8_e4m3fn).double().t()
            y += part * s["xs"][k // BLOCK].double()[:, None] * s["ws"][:, k // BLOCK].double().repeat_interleave(BLOCK)[: c["N"]]
        return y if s["b"] is None else y + s["b"].double()
    ql, kl = _lengths(c)
    D, group = c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros((sum(ql), c["heads"] * D), dtype=torch.float64, device="cuda")
    r0, begin = 0, s["begin"].tolist()
    for b in range(c["B"]):
        for h in range(c["heads"] if kl[b] else 0):
            j = (h // group) * D
            K = s["kv"][begin[b] : begin[b] + kl[b], j : j + D].double()
            V = s["kv"][begin[b] : begin[b] + kl[b], (c["kv_heads"] * D) + j : (c["kv_heads"] * D) + j + D].double()
            out[r0 : r0 + ql[b], h * D : (h + 1) * D] = torch.softmax(s["q"][r0 : r0 + ql[b], h * D : (h + 1) * D].double() @ K.t() / math.sqrt(D), 1) @ V
        r0 += ql[b]
    return out
