"""choreo_quantize_block and choreo_gemm_block_scaled against plain
restatements of their definitions.

Quantisation is exact: scales and e4m3 values equal the definition's bit for
bit. Products are compared with 64-bit sums of the dequantised operands. For
each element, with S = sum over k of |a b| (scales included),
  - the products of two e4m3 values (4 significant bits each) are exact in
    fp32; the tensor cores add 128 of them per block in steps of 32, each step
    and each of the alignments in it off by at most 2^-23 of the block's sum
    of magnitudes: (128 / 32 + 2) steps;
  - each block's scale product, scaling and addition to the running sum rounds
    by 2^-24 each of what is summed: 3 per block, at most K/128 + 3 of them;
  - alpha, the addend and the bias add a rounding of 2^-24 each of the
    magnitudes they meet;
  - the store rounds by half a step of the output type.
"""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

F8 = "float8_e4m3fn"


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def quantize_plain(x, block_rows, transpose):
    """The definition on the host, every step rounded to fp32."""
    import torch
    x = x.detach().cpu().float()
    if transpose:
        x = x.t()
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    full = torch.zeros(rb * block_rows, cb * 128)
    full[:rows, :cols] = x
    parts = full.view(rb, block_rows, cb, 128)
    mag = parts.abs()
    mag = torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag))
    amax = mag.amax(dim=(1, 3)).clamp_min(2.0 ** -100)
    top = torch.full_like(amax, 448.0)
    inv, scale = top / amax, amax / top
    v = torch.where(torch.isfinite(parts), parts, torch.full_like(parts, float("nan"))) * inv[:, None, :, None]
    return v.reshape(full.shape)[:rows, :cols].to(torch.float8_e4m3fn), scale


def run_quantize(cb, x, block_rows, transpose, *, pad_q=0, scale_major="k"):
    import torch
    r, c = (x.shape[1], x.shape[0]) if transpose else tuple(x.shape)
    ldq = c + pad_q
    q = torch.full((r + 1, ldq), 0x55, dtype=torch.uint8, device="cuda")
    rb, kb = -(-r // block_rows), -(-c // 128)
    store = torch.full((kb + 1, rb + 1) if scale_major == "k" else (rb + 1, kb + 1), -7.0, device="cuda")
    scale = store[:kb, :rb].t() if scale_major == "k" else store[:rb, :kb]
    cb.quantize_block(x, q[:r, :c], scale, block_rows=block_rows, transpose=transpose)
    cb.sync_status()
    # nothing behind the rows, the columns or the scales is written
    assert (q[r:] == 0x55).all() and (q[:, c:] == 0x55).all()
    assert (store[-1] == -7.0).all() and (store[:, -1] == -7.0).all()
    return q[:r, :c].contiguous().view(torch.float8_e4m3fn), scale


def same_e4m3(a, b):
    import torch
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    nan_a, nan_b = (a & 0x7F) == 0x7F, (b & 0x7F) == 0x7F
    return torch.equal(nan_a, nan_b) and torch.equal(a[~nan_a], b[~nan_b])


SHAPES = [(1, 1), (1, 128), (3, 127), (13, 4096), (128, 128), (129, 257), (300, 1000), (517, 2064), (8, 5000)]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_equals_definition(cb, cuda, dt, block_rows, transpose):
    import torch
    for i, (rows, cols) in enumerate(SHAPES):
        g = torch.Generator(device="cuda")
        g.manual_seed(100 + i)
        pad = (8 - cols % 8) % 8 if i % 2 == 0 else 3   # 16-byte aligned rows, and rows at any offset
        x = torch.randn(rows, cols + pad, generator=g, device="cuda")
        x *= torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g, device="cuda").float())
        x = x.to(_dt(dt))[:, :cols]
        q, scale = run_quantize(cb, x, block_rows, transpose, pad_q=(16 - q_cols(x, transpose) % 16) % 16 if i % 3 else 1,
                                scale_major="k" if i % 2 else "row")
        want_q, want_s = quantize_plain(x, block_rows, transpose)
        assert torch.equal(scale.cpu(), want_s), (rows, cols)
        assert same_e4m3(q, want_q), (rows, cols)


def q_cols(x, transpose):
    return x.shape[0] if transpose else x.shape[1]


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("pad", [0, 1])
def test_quantize_special_values(cb, cuda, dt, block_rows, transpose, pad):
    """Zero blocks, subnormals, NaN and infinities (which leave their block's
    scale alone), the type's largest values, ties."""
    import torch
    t = _dt(dt)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    x = torch.randn(264, 512 + pad, generator=g, device="cuda").to(t)[:, :512]
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 200] = float("-inf")
    x[3, 300:310] = float("nan")
    x[4, :128] = float("nan")
    x[5] = torch.finfo(t).max
    x[6] = torch.finfo(t).tiny
    x[7] = torch.finfo(t).smallest_normal / 4
    x[8, :128] = torch.arange(128, device="cuda").to(t) * 3.5   # ties: 3.5 * 2^k multiples of a 448 maximum
    x[8, 127] = 448.0
    x[130:200, 128:256] = float("inf")
    q, scale = run_quantize(cb, x, block_rows, transpose)
    want_q, want_s = quantize_plain(x, block_rows, transpose)
    assert torch.equal(scale.cpu(), want_s)
    assert same_e4m3(q, want_q)


def test_quantize_empty_is_a_no_op(cb, cuda):
    import ctypes as C
    for rows, cols in ((0, 5), (5, 0), (0, 0)):
        d = cb.QuantDesc()
        d.rows, d.cols, d.dtype, d.block_rows = rows, cols, cb.BF16, 1
        assert cb.lib.choreo_quantize_block(C.byref(d), None) == cb.OK


def test_quantize_many_rows(cb, cuda):
    """More row tiles than a launch dimension of 65535 holds."""
    import torch
    rows = 65537 * 128 + 5
    x = torch.ones(rows, 8, device="cuda", dtype=torch.bfloat16)
    x[-1] = 2
    for block_rows, transpose in ((1, False), (128, False), (128, True)):
        r, c = (8, rows) if transpose else (rows, 8)
        q = torch.empty(r, c, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        scale = torch.empty(-(-c // 128), -(-r // block_rows), device="cuda").t()
        cb.quantize_block(x, q, scale, block_rows=block_rows, transpose=transpose)
        cb.sync_status()
        back = q.float() * (scale.repeat_interleave(128, 1)[:, :c].repeat_interleave(block_rows, 0)[:r])
        want = x.t() if transpose else x
        assert torch.equal(back, want.float())


# ------------------------------------------------------------------ product
def make_operand(cb, rows, k, seed, block, std=1.0, pad=0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda") * std
    loud = torch.rand(k, generator=g, device="cuda") < 0.02
    x = x * torch.where(loud, 20.0, 1.0)
    ld = -(-k // 16) * 16 + pad
    q8, scale = quantize_plain(x, block, False)
    q = torch.full((rows, ld), 0x7F, dtype=torch.uint8, device="cuda")  # NaN behind the rows: never read
    q[:, :k] = q8.view(torch.uint8).cuda()
    return q.view(torch.float8_e4m3fn)[:, :k], scale.cuda()


def dequantize(q, scale, block):
    full = scale.double().repeat_interleave(128, 1)[:, : q.shape[1]]
    return q.float().double() * full.repeat_interleave(block, 0)[: q.shape[0]]


def product_and_bound(a, sa, b, sb, block_b, out_dt, *, alpha=1.0, beta=0.0, addend=None, bias=None, relu=False):
    import torch
    da, db = dequantize(a, sa, 1), dequantize(b, sb, block_b)
    want, mag = da @ db.t(), da.abs() @ db.abs().t()
    blocks = -(-a.shape[1] // 128)
    err = ((128 // 32 + 2) * 2.0 ** -23 + (blocks + 3) * 2.0 ** -24) * mag
    want, err = want * alpha, err * abs(alpha) + 2.0 ** -24 * mag * abs(alpha)
    if addend is not None:
        want = want + beta * addend.double()
        err = err + 2.0 ** -24 * ((beta * addend.double()).abs() + want.abs()) * 2
    if bias is not None:
        want = want + bias.double()
        err = err + 2.0 ** -24 * (bias.double().abs() + want.abs())
    if relu:
        want = want.clamp_min(0)
    eps = torch.finfo(out_dt).eps
    tiny = torch.finfo(out_dt).smallest_normal * eps  # half a step below the normal numbers, doubled
    return want, err * (1 + eps) + eps / 2 * want.abs() + tiny


def assert_within(got, want, bound, what):
    import torch
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs()
    assert (off <= bound).all(), (what, (off / bound).max().item())


GEMM_SHAPES = [(1, 1, 1), (1, 128, 128), (1, 300, 4096), (7, 129, 100), (16, 256, 1000), (31, 1000, 384),
               (64, 64, 2048), (65, 200, 129), (128, 128, 128), (129, 257, 511), (200, 1031, 777), (300, 129, 5000),
               (1031, 2053, 1999), (2048, 1280, 256)]


@pytest.mark.parametrize("block_b", [1, 128])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
def test_product_against_64_bits(cb, cuda, block_b, out):
    import torch
    for i, (m, n, k) in enumerate(GEMM_SHAPES):
        a, sa = make_operand(cb, m, k, 10 + i, 1, pad=16 * (i % 3))
        b, sb = make_operand(cb, n, k, 90 + i, block_b, std=k ** -0.5)
        if i % 2:   # the layout the kernel reads fastest, and the other one
            sa, sb = sa.t().contiguous().t(), sb.t().contiguous().t()
        ldc = n if i % 2 else -(-n // 8) * 8 + 8
        c = torch.full((m + 1, ldc), 5.0, device="cuda", dtype=_dt(out))
        cb.gemm_block_scaled(a, sa, b, sb, c[:m, :n])
        cb.sync_status()
        want, bound = product_and_bound(a, sa, b, sb, block_b, _dt(out))
        assert_within(c[:m, :n], want, bound, (m, n, k))
        assert (c[m:] == 5.0).all() and (c[:, n:] == 5.0).all()


@pytest.mark.parametrize("m", [1, 20, 64, 66, 96, 128])
@pytest.mark.parametrize("block_b", [1, 128])
def test_few_rows_in_every_number_of_pieces(cb, cuda, block_b, m):
    import torch
    seen = set()
    for tiles, k in ((160, 200), (120, 1100), (80, 1600), (60, 2100), (45, 2700), (40, 3200), (35, 3800), (20, 4100)):
        n = 128 * tiles - 3
        a, sa = make_operand(cb, m, k, 10, 1)
        b, sb = make_operand(cb, n, k, 90, block_b, std=k ** -0.5)
        c = torch.full((m + 1, n), 5.0, device="cuda", dtype=torch.float32)
        seen.add(cb.gemm_block_scaled_query(cb.gemm_block_desc(a, sa, b, sb, c[:m])).split_k)
        cb.gemm_block_scaled(a, sa, b, sb, c[:m])
        cb.sync_status()
        want, bound = product_and_bound(a, sa, b, sb, block_b, torch.float32)
        assert_within(c[:m], want, bound, (m, n, k))
        assert (c[m:] == 5.0).all()
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert seen == set(range(1, 9))


@pytest.mark.parametrize("m,n,k", [(5, 300, 1000), (200, 264, 700), (1100, 1288, 900)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("block_b", [1, 128])
def test_product_epilogue(cb, cuda, m, n, k, out, block_b):
    """alpha, beta with an addend of its own stride and in place, bias, ReLU."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    a, sa = make_operand(cb, m, k, 1, 1)
    b, sb = make_operand(cb, n, k, 2, block_b, std=k ** -0.5)
    t = _dt(out)
    for ldd in (n, n + 3):
        addend = torch.randn(m, ldd, generator=g, device="cuda").to(t)[:, :n]
        bias = torch.randn(n, generator=g, device="cuda").to(torch.bfloat16)
        c = torch.empty(m, n, device="cuda", dtype=t)
        cb.gemm_block_scaled(a, sa, b, sb, c, alpha=0.5, beta=-1.5, addend=addend, bias=bias, relu=True)
        cb.sync_status()
        want, bound = product_and_bound(a, sa, b, sb, block_b, t, alpha=0.5, beta=-1.5, addend=addend, bias=bias,
                                        relu=True)
        assert_within(c, want, bound, "addend")
        c.copy_(addend)
        cb.gemm_block_scaled(a, sa, b, sb, c, beta=1.0)
        cb.sync_status()
        want, bound = product_and_bound(a, sa, b, sb, block_b, t, beta=1.0, addend=addend)
        assert_within(c, want, bound, "in place")
    # beta == 0 reads neither C nor the addend
    c.fill_(float("nan"))
    cb.gemm_block_scaled(a, sa, b, sb, c, addend=torch.full_like(c, float("nan")))
    cb.sync_status()
    want, bound = product_and_bound(a, sa, b, sb, block_b, t)
    assert_within(c, want, bound, "beta 0")


@pytest.mark.parametrize("m,n,k", [(3, 200, 500), (700, 900, 640)])
def test_product_nan_stays_in_its_row_and_column(cb, cuda, m, n, k):
    import torch
    a, sa = make_operand(cb, m, k, 1, 1)
    b, sb = make_operand(cb, n, k, 2, 128)
    ref = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    cb.gemm_block_scaled(a, sa, b, sb, ref)
    a.view(torch.uint8)[1, 77] = 0x7F
    b.view(torch.uint8)[150, 3] = 0xFF
    c = torch.empty_like(ref)
    cb.gemm_block_scaled(a, sa, b, sb, c)
    cb.sync_status()
    nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    nan[1], nan[:, 150] = True, True
    assert torch.equal(torch.isnan(c), nan)
    assert torch.equal(c[~nan], ref[~nan])


@pytest.mark.parametrize("m,n,k", [(4, 512, 4096), (100, 1000, 900), (1500, 2000, 1100)])
def test_product_repeats_bit_for_bit_in_a_graph(cb, cuda, m, n, k):
    import torch
    a, sa = make_operand(cb, m, k, 1, 1)
    b, sb = make_operand(cb, n, k, 2, 128)
    ref = torch.empty(m, n, device="cuda", dtype=torch.float32)
    cb.gemm_block_scaled(a, sa, b, sb, ref)
    cb.sync_status()
    c = torch.empty_like(ref)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cb.gemm_block_scaled(a, sa, b, sb, c)   # warm-up on the capture's stream
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            cb.gemm_block_scaled(a, sa, b, sb, c)
    for _ in range(3):
        c.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, ref)


@pytest.mark.parametrize("m,n,k", [(1, 200, 1001), (150, 1, 333), (1, 1, 5)])
def test_product_of_a_single_row(cb, cuda, m, n, k):
    """One row's length is free: it starts on a 16-byte boundary by itself."""
    import torch
    a, sa = make_operand(cb, m, k, 1, 1)
    b, sb = make_operand(cb, n, k, 2, 1)
    if m == 1:
        a = a.view(torch.uint8).flatten().clone().view(1, k)
    if n == 1:
        b = b.view(torch.uint8).flatten().clone().view(1, k)
    c = torch.empty(m, n, device="cuda")
    cb.gemm_block_scaled(a, sa, b, sb, c)
    cb.sync_status()
    want, bound = product_and_bound(a.view(torch.float8_e4m3fn), sa, b.view(torch.float8_e4m3fn), sb, 1, torch.float32)
    assert_within(c, want, bound, (m, n, k))


@pytest.mark.parametrize("m", [100, 300])
def test_offsets_past_32_bits(cb, cuda, m):
    """Rows 2^23 elements apart, of the values, codes, scales and outputs."""
    import torch
    n, k, ld = 264, 500, 1 << 23
    x = torch.randn(300, k, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    floats = torch.empty(300, ld, device="cuda")
    codes = torch.empty(k, ld, dtype=torch.uint8, device="cuda")
    floats[:, :k] = x
    for block, trans in ((1, False), (128, False), (1, True), (128, True)):
        r, c = (k, 300) if trans else (300, k)
        q, want_q = codes[:r, :c].view(torch.float8_e4m3fn), torch.empty(r, -(-c // 16) * 16, dtype=torch.uint8, device="cuda")
        want_q = want_q[:, :c].view(torch.float8_e4m3fn)
        rows = -(-r // block)
        scale = floats[:rows, 1024:1024 + -(-c // 128)] if rows <= 300 else torch.empty(rows, -(-c // 128), device="cuda")
        want_s = torch.empty(rows, -(-c // 128), device="cuda")
        cb.quantize_block(floats[:, :k], q, scale, block_rows=block, transpose=trans)
        cb.quantize_block(x, want_q, want_s, block_rows=block, transpose=trans)
        cb.sync_status()
        assert torch.equal(scale, want_s) and torch.equal(q.contiguous().view(torch.uint8), want_q.contiguous().view(torch.uint8))
    for block_b in (1, 128):
        a, sa = make_operand(cb, m, k, 1, 1)
        b, sb = make_operand(cb, n, k, 2, block_b)
        addend = torch.randn(m, n, device="cuda")
        fa, fb = codes[:m, :k], codes[:n, 1024:1024 + k]
        fa.copy_(a.view(torch.uint8))
        fb.copy_(b.view(torch.uint8))
        fsa, fsb = floats[:m, 2048:2052], floats[:sb.shape[0], 2064:2068]
        fsa.copy_(sa)
        fsb.copy_(sb)
        d, c, near = floats[:m, 4096:4096 + n], floats[:m, 8192:8192 + n], torch.empty(m, n, device="cuda")
        d.copy_(addend)
        cb.gemm_block_scaled(fa.view(torch.float8_e4m3fn), fsa, fb.view(torch.float8_e4m3fn), fsb, c, beta=2.0, addend=d)
        cb.gemm_block_scaled(a, sa, b, sb, near, beta=2.0, addend=addend)
        cb.sync_status()
        assert torch.equal(c, near)


def test_quantize_then_product(cb, cuda):
    """The three products of a linear layer in 8 bits: forward, input gradient
    (the weight quantised transposed) and weight gradient (both operands along
    the tokens, added to an f32 sum)."""
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    m, n, k = 300, 520, 648
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    dy = torch.randn(m, n, generator=g, device="cuda").bfloat16()

    def quant(t, block, transpose=False):
        r, c = (t.shape[1], t.shape[0]) if transpose else tuple(t.shape)
        q = torch.empty(r, -(-c // 16) * 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :c]
        scale = torch.empty(-(-c // 128), -(-r // block), device="cuda").t()
        cb.quantize_block(t, q, scale, block_rows=block, transpose=transpose)
        return q, scale

    for a, b, block_b, shape, dt in (
            (quant(x, 1), quant(w, 128), 128, (m, n), torch.bfloat16),
            (quant(dy, 1), quant(w, 128, True), 128, (m, k), torch.bfloat16),
            (quant(dy, 1, True), quant(x, 1, True), 1, (n, k), torch.float32)):
        start = torch.randn(shape, generator=g, device="cuda").to(dt)
        c = start.clone()
        cb.gemm_block_scaled(*a, *b, c, beta=1.0)
        cb.sync_status()
        want, bound = product_and_bound(*a, *b, block_b, dt, beta=1.0, addend=start)
        assert_within(c, want, bound, shape)
