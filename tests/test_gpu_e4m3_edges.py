"""The e4m3 path where it can go wrong beyond its ordinary shapes: rows of more than 2^31 bytes."""

import numpy as np
import pytest

import e4m3_reference as ref
from test_gpu_e4m3 import DT, call, status, tdt

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
