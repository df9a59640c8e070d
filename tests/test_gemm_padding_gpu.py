"""choreo_gemm leaves what lies behind C's rows alone, whatever N and the
leading dimension: a C that is a window of a larger matrix keeps its
neighbours, and padding keeps its contents."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile", ["", "wide256", "pair256", "pair128", "single256", "single128", "single64"])
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(3, 5, 64), (300, 13, 64), (700, 1003, 128), (130, 262, 96)])
def test_columns_behind_n_are_untouched(cb, cuda, tile, out, m, n, k):
    import torch
    dt = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[out]
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    a = torch.randint(-4, 5, (m, k), generator=g, device="cuda").half()
    b = torch.randint(-4, 5, (k, -(-n // 8) * 8), generator=g, device="cuda").half()[:, :n]
    if dt == torch.bfloat16:
        a, b = a.bfloat16(), b.bfloat16()
    buf = torch.full((m + 2, -(-n // 8) * 8 + 8), 5.0, device="cuda", dtype=dt)
    with cb.tuning(tile=tile):
        cb.gemm(a, b, buf[1:m + 1, :n])
    cb.sync_status()
    want = (a.double() @ b.double()).to(dt)  # whole numbers below 2^11: exact in fp32
    assert torch.equal(buf[1:m + 1, :n], want)
    assert (buf[:, n:] == 5.0).all() and (buf[0] == 5.0).all() and (buf[m + 1] == 5.0).all()
