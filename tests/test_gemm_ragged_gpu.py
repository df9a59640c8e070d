"""choreo_gemm and the weight gradients where the rows of a padded output end
inside 16 bytes: whole groups of columns go out as bulk tensor stores, the last
one element by element, and nothing behind the rows changes."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

TILES = ["", "wide256", "pair256", "pair128", "single256", "single128", "single64"]


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def whole(rows, cols, dt, seed, pad=0, top=3):
    """Whole numbers in -top .. top: sums below 2^11 are exact in every type used here."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(-top, top + 1, (rows, cols + pad), generator=g, device="cuda").to(dt)[:, :cols]


def window(m, n, dt, fill):
    """An m x n window with 16-byte aligned rows that continue behind it, and a row before and after."""
    import torch
    ld = -(-n // 8) * 8 + 8
    buf = torch.full((m + 2, ld), fill, device="cuda", dtype=dt)
    return buf[1:m + 1, :n], buf


def kept(buf, m, n, fill):
    return bool((buf[:, n:] == fill).all() and (buf[0] == fill).all() and (buf[m + 1] == fill).all())


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("beta,bias,relu", [(0.0, False, False), (0.0, True, True), (1.0, True, False)])
def test_every_tail(cb, cuda, tile, out, beta, bias, relu):
    """N that ends 1 .. 63 columns into a group, in the first tile's columns and
    behind whole tiles; rows that end inside a warp's 32."""
    import torch
    dt = _dt(out)
    ab = torch.bfloat16 if out == "bf16" else torch.float16
    for i, n in enumerate((1, 7, 9, 31, 33, 63, 65, 95, 127, 129, 190, 255, 257, 319, 447, 513, 517)):
        m, k = (5, 129, 300, 545)[i % 4], 40   # products below 9 * 40 + 6 < 2^9: exact
        a, b = whole(m, k, ab, n), whole(k, n, ab, n + 1, pad=-n % 8)
        c, buf = window(m, n, dt, 2.0)
        vec = whole(1, n, torch.float32, 5)[0].contiguous() if bias else None
        want = a.double() @ b.double() + (2.0 * beta) + (vec.double() if bias else 0.0)
        if relu:
            want = want.clamp_min(0)
        if out == "bf16":
            want = want.to(dt).double()
        with cb.tuning(tile=tile):
            cb.gemm(a, b, c, beta=beta, bias=vec, relu=relu)
        cb.sync_status()
        assert torch.equal(c.double(), want), (n, m)
        assert kept(buf, m, n, 2.0), (n, m)


@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("trans_b", [False, True])
def test_batches_and_split_sums(cb, cuda, out, trans_b):
    """Batch items of a padded output, and K cut into ranges (the partial sums
    are rows of N f32 without padding)."""
    import torch
    dt = _dt(out)
    for n in (13, 130, 201):
        a = torch.stack([whole(70, 64, torch.float16, s) for s in range(3)])
        b = torch.stack([whole(n, 64, torch.float16, 9 + s) if trans_b else whole(64, -(-n // 8) * 8, torch.float16, 9 + s)
                         for s in range(3)])
        b = b if trans_b else b[:, :, :n]
        ld = -(-n // 8) * 8
        buf = torch.full((3, 71, ld), 4.0, device="cuda", dtype=dt)
        cb.gemm(a, b, buf[:, :70, :n], trans_b=trans_b)
        cb.sync_status()
        want = a.double() @ (b.double().transpose(1, 2) if trans_b else b.double())
        assert torch.equal(buf[:, :70, :n].double(), want)
        assert (buf[:, :, n:] == 4.0).all() and (buf[:, 70] == 4.0).all()
        a1, b1 = whole(33, 1024, torch.float16, n, top=1), whole(1024, n, torch.float16, n + 1, pad=-n % 8, top=1)
        c, cbuf = window(33, n, dt, 2.0)
        with cb.tuning(split_k=2):
            cb.gemm(a1, b1, c)
        cb.sync_status()
        assert torch.equal(c.double(), a1.double() @ b1.double()) and kept(cbuf, 33, n, 2.0)


@pytest.mark.parametrize("tile", ["", "wide256", "pair256", "single128"])
@pytest.mark.parametrize("dw", ["bf16", "f32"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weight_gradients_of_odd_width(cb, cuda, tile, dw, accumulate):
    """Weights K x N with an odd N and padded rows, and dX with an odd K: equal
    to the same call on contiguous N x K storage to the bit (the sums run in the
    same order), and nothing behind the rows changes."""
    import torch
    for m, n, k in ((200, 101, 75), (90, 517, 300)):
        g = torch.Generator(device="cuda")
        g.manual_seed(n)

        def rand(rows, cols, std):
            return (torch.randn(rows, cols + -cols % 8, generator=g, device="cuda") * std).bfloat16()[:, :cols]

        x, dh, wg, wu = rand(m, k, 1.0), rand(m, n, 0.5), rand(k, n, k ** -0.5), rand(k, n, k ** -0.5)
        dt = _dt(dw)
        dwg, gbuf = window(k, n, dt, 2.0)
        dwu, ubuf = window(k, n, dt, 2.0)
        dx, xbuf = window(m, k, torch.bfloat16, 2.0)
        flat = [torch.full((n, k), 2.0, device="cuda", dtype=dt) for _ in range(2)]
        flat_dx = torch.empty(m, k, device="cuda", dtype=torch.bfloat16)
        with cb.tuning(tile=tile):
            cb.gated_ffn_backward(dh, x, wg, wu, dx=dx, dw_gate=dwg, dw_up=dwu, accumulate=accumulate)
            cb.gated_ffn_backward(dh, x, wg.t().contiguous(), wu.t().contiguous(), dx=flat_dx, dw_gate=flat[0],
                                  dw_up=flat[1], trans_w=True, accumulate=accumulate)
        cb.sync_status()
        assert torch.equal(dwg, flat[0].t()) and torch.equal(dwu, flat[1].t()) and torch.equal(dx, flat_dx)
        assert kept(gbuf, k, n, 2.0) and kept(ubuf, k, n, 2.0) and kept(xbuf, m, k, 2.0)
