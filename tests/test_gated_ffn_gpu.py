"""choreo_gated_ffn and its backward pass against the formulas in 64 bits.

Bounds, element by element, with u = 2^-24 and eps the 16-bit type's step:
  - a product summed over L elements by the tensor cores in fp32 (16 per step,
    a step off by at most 2 u of the sum of magnitudes so far, plus 4 for the
    joins of split sums): (L / 16 + 4) 2 u S, S = sum of |a b|;
  - an activation value or slope: 2^-16 of |g| + |value| covers the exponential,
    the divisions and the polynomial of the kernel's formulas (2e-5 at most, far
    out in the tail of GELU);
  - every store in 16 bits rounds by eps / 2 of the value, or half of the
    smallest subnormal step;
  - what is computed from such values carries their bounds through the formula.
"""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu"]
U = 2.0 ** -24


def _dt(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def act64(g, act):
    """The activation and its slope in 64 bits."""
    import torch
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        phi = torch.special.ndtr(g)
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    return g.clamp_min(0), (g > 0).double()


def rounding(v, dt):
    import torch
    f = torch.finfo(dt)
    return f.eps / 2 * v.abs() + f.smallest_normal * f.eps / 2


def sum_bound(mag, length):
    return (length / 16 + 4) * 2 * U * mag


def matrix(rows, cols, dt, seed, std=1.0, pad=0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    m = torch.full((rows, cols + pad), float("nan"), device="cuda", dtype=dt)  # NaN behind the rows: never read
    m[:, :cols] = (torch.randn(rows, cols, generator=g, device="cuda") * std).to(dt)
    return m[:, :cols]


def output(rows, cols, dt, pad=0):
    """A view with padding and a row behind it that must not change."""
    import torch
    buf = torch.full((rows + 1, cols + pad), 3.0, device="cuda", dtype=dt)
    return buf[:rows, :cols], buf


def untouched(buf, rows, cols):
    return bool((buf[rows:] == 3.0).all() and (buf[:, cols:] == 3.0).all())


def assert_within(got, want, bound, what):
    import torch
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item()
    assert (off <= bound).all(), (what, worst)


class Case:
    def __init__(self, m, n, k, dt, act, trans, *, pads=(0, 0, 0), seed=0, scale=1.0):
        self.m, self.n, self.k, self.act, self.trans = m, n, k, act, trans
        self.dt = _dt(dt)
        self.x = matrix(m, k, self.dt, seed + 1, scale, pads[0])
        shape = (n, k) if trans else (k, n)
        self.wg = matrix(*shape, self.dt, seed + 2, k ** -0.5, pads[1])
        self.wu = matrix(*shape, self.dt, seed + 3, k ** -0.5, pads[1])
        self.dh = matrix(m, n, self.dt, seed + 4, 0.5, pads[2])
        self.wgd = self.wg.double().t() if trans else self.wg.double()   # K x N
        self.wud = self.wu.double().t() if trans else self.wu.double()

    def products(self):
        """G, U and their bounds."""
        x = self.x.double()
        g, u = x @ self.wgd, x @ self.wud
        return (g, u, sum_bound(x.abs() @ self.wgd.abs(), self.k), sum_bound(x.abs() @ self.wud.abs(), self.k))

    def hidden(self, g, u, eg, eu):
        """H and its bound before the store."""
        v, dv = act64(g, self.act)
        ev = 1.2 * eg + 2.0 ** -16 * (v.abs() + g.abs() * 1e-3)
        return v * u, (v.abs() + ev) * eu + ev * u.abs()


SHAPES = [  # m, n, k, pads of x, w and outputs: aligned rows and rows at any offset
    (1, 1, 1, (0, 0, 0)), (1, 64, 64, (0, 0, 0)), (1, 200, 4096, (0, 0, 0)), (3, 129, 72, (1, 3, 5)),
    (16, 2000, 264, (0, 0, 8)), (17, 65, 1000, (0, 0, 0)), (33, 640, 96, (8, 8, 8)), (64, 130, 520, (0, 2, 0)),
    (65, 257, 136, (0, 0, 0)), (128, 64, 2048, (0, 0, 0)), (129, 321, 200, (0, 7, 1)), (257, 515, 333, (3, 5, 1)),
    (700, 1000, 128, (0, 0, 0)), (1030, 1290, 264, (0, 0, 6)),
]


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
def test_forward(cb, cuda, trans, dt, act):
    for i, (m, n, k, pads) in enumerate(SHAPES):
        c = Case(m, n, k, dt, act, trans, pads=pads, seed=10 * i)
        h, hbuf = output(m, n, c.dt, pads[2])
        keep = i % 2 == 0
        gate, gbuf = output(m, n, c.dt, pads[2]) if keep else (None, None)
        up, ubuf = output(m, n, c.dt, pads[2]) if keep else (None, None)
        cb.gated_ffn(c.x, c.wg, c.wu, h, act=act, trans_w=trans, gate=gate, up=up)
        cb.sync_status()
        g, u, eg, eu = c.products()
        want, e = c.hidden(g, u, eg, eu)
        assert_within(h, want, e + rounding(want.abs() + e, c.dt), ("h", m, n, k))
        assert untouched(hbuf, m, n), (m, n, k)
        if keep:
            assert_within(gate, g, eg + rounding(g.abs() + eg, c.dt), ("gate", m, n, k))
            assert_within(up, u, eu + rounding(u.abs() + eu, c.dt), ("up", m, n, k))
            assert untouched(gbuf, m, n) and untouched(ubuf, m, n)


@pytest.mark.parametrize("m", [1, 5, 17, 50, 77, 96, 97, 128])
@pytest.mark.parametrize("trans", [False, True])
def test_few_rows_in_every_number_of_pieces(cb, cuda, trans, m):
    """K is cut over one to eight CTAs, unevenly where it does not divide; a
    rank may have no row of H to add up."""
    seen = set()
    for tiles, k in ((300, 100), (120, 700), (80, 1000), (60, 1300), (45, 1400), (40, 1610), (35, 1900), (20, 2100)):
        n = 64 * tiles - 3
        c = Case(m, n, k, "bf16", "silu", trans, seed=tiles)
        h, hbuf = output(m, n, c.dt, 1)
        q = cb.gated_ffn_query(cb.ffn_desc(c.x, c.wg, c.wu, h, trans_w=trans))
        seen.add(q.split_k)
        # a ring of `stages` k-blocks of 128 weight rows and tile_m tokens, 128 bytes each, and under 2 KB besides
        assert m <= q.tile_m <= 128 and q.tmem_cols == max(32, 1 << (q.tile_m - 1).bit_length())
        assert 0 < q.smem_bytes - q.stages * (128 + q.tile_m) * 128 < 2048
        cb.gated_ffn(c.x, c.wg, c.wu, h, trans_w=trans)
        cb.sync_status()
        g, u, eg, eu = c.products()
        want, e = c.hidden(g, u, eg, eu)
        assert_within(h, want, e + rounding(want.abs() + e, c.dt), (m, tiles))
        assert untouched(hbuf, m, n), (m, tiles)
    if cuda_sms() == 148:
        assert seen == set(range(1, 9))


def cuda_sms():
    import torch
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("tile", ["wide256", "pair256", "single128"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_forward_and_backward_every_tile(cb, cuda, tile, trans, act):
    with cb.tuning(tile=tile):
        for m, n, k in ((130, 200, 200), (600, 390, 1032)):
            c = Case(m, n, k, "bf16", act, trans)
            h, hbuf = output(m, n, c.dt, 2)
            cb.gated_ffn(c.x, c.wg, c.wu, h, act=act, trans_w=trans)
            cb.sync_status()
            g, u, eg, eu = c.products()
            want, e = c.hidden(g, u, eg, eu)
            assert_within(h, want, e + rounding(want.abs() + e, c.dt), (tile, m))
            assert untouched(hbuf, m, n)
            check_backward(cb, c, False, "f32", False, 1, (tile, m))
            check_backward(cb, c, True, "bf16", True, 0, (tile, m))


def check_backward(cb, c, keep, dw_name, accumulate, pad, what, *, want_dx=True, want_dw=True, want_h=True):
    """Runs the backward pass and checks every output and what lies behind it."""
    import torch
    m, n, k, dt = c.m, c.n, c.k, c.dt
    g, u, eg, eu = c.products()
    gate = up = None
    if keep:
        gate, up = g.to(dt), u.to(dt)
        g, u = gate.double(), up.double()
        eg = eu = torch.zeros_like(g)
    dw_dt = _dt(dw_name)
    wshape = (n, k) if c.trans else (k, n)
    dx, dxbuf = output(m, k, dt, pad) if want_dx else (None, None)
    dwg, dwgbuf = output(*wshape, dw_dt, pad) if want_dw else (None, None)
    dwu, dwubuf = output(*wshape, dw_dt, pad) if want_dw else (None, None)
    h, hbuf = output(m, n, dt, pad) if want_h else (None, None)
    cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=dx, dw_gate=dwg, dw_up=dwu, gate=gate, up=up, h=h, act=c.act,
                          trans_w=c.trans, accumulate=accumulate)
    cb.sync_status()
    dh = c.dh.double()
    v, dv = act64(g, c.act)
    ev = 1.2 * eg + 2.0 ** -16 * (v.abs() + g.abs() * 1e-3)
    # slopes of the slopes are below 1.2 too; ReLU's slope jumps where G is within its bound of 0
    edv = 1.2 * eg + 2.0 ** -16 * (dv.abs() + 1e-3)
    if c.act == "relu":
        edv = torch.where(g.abs() <= eg, torch.ones_like(g), edv)
    dg, du = dh * u * dv, dh * v
    edg = dh.abs() * ((u.abs() + eu) * edv + eu * dv.abs()) + 4 * U * dg.abs()
    edu = dh.abs() * ev + 2 * U * du.abs()
    edg, edu = edg + rounding(dg.abs() + edg, dt), edu + rounding(du.abs() + edu, dt)
    if want_h:
        hw, he = c.hidden(g, u, eg, eu)
        assert_within(h, hw, he + rounding(hw.abs() + he, dt), ("h", what))
        assert untouched(hbuf, m, n), what
    if want_dx:
        want = dg @ c.wgd.t() + du @ c.wud.t()
        mag = (dg.abs() + edg) @ c.wgd.abs().t() + (du.abs() + edu) @ c.wud.abs().t()
        e = edg @ c.wgd.abs().t() + edu @ c.wud.abs().t() + sum_bound(mag, 2 * n)
        assert_within(dx, want, e + rounding(want.abs() + e, dt), ("dx", what))
        assert untouched(dxbuf, m, k), what
    if want_dw:
        x = c.x.double()
        for got, buf, d, ed, name in ((dwg, dwgbuf, dg, edg, "dw_gate"), (dwu, dwubuf, du, edu, "dw_up")):
            want = x.t() @ d
            e = x.abs().t() @ ed + sum_bound(x.abs().t() @ (d.abs() + ed), m)
            if c.trans:
                want, e = want.t(), e.t()
            if accumulate:
                want = want + 3.0   # what output() filled the matrix with
                e = e + 2 * U * (want.abs() + 3.0)
            assert_within(got, want, e + rounding(want.abs() + e, dw_dt), (name, what))
            assert untouched(buf, *wshape), (name, what)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [False, True])
def test_backward(cb, cuda, trans, dt, act, keep):
    for i, (m, n, k, pads) in enumerate(SHAPES):
        c = Case(m, n, k, dt, act, trans, pads=pads, seed=10 * i)
        check_backward(cb, c, keep, dt if i % 2 else "f32", i % 3 == 1, pads[2], (m, n, k), want_h=i % 2 == 0)


@pytest.mark.parametrize("keep", [False, True])
def test_backward_parts(cb, cuda, keep):
    c = Case(150, 264, 320, "bf16", "silu", False)
    check_backward(cb, c, keep, "f32", False, 0, "dx alone", want_dw=False, want_h=False)
    check_backward(cb, c, keep, "f32", False, 0, "dw alone", want_dx=False, want_h=False)


@pytest.mark.parametrize("m,n,k", [(40, 8192, 256), (200, 4096, 128)])
def test_backward_split_sum(cb, cuda, m, n, k):
    """Few output tiles over a long 2 N sum: dX is split over K ranges when the
    workspace holds the partial sums, and the same call without them is not."""
    import ctypes as C
    import torch
    c = Case(m, n, k, "bf16", "silu", True)
    d = cb.ffn_grad_desc(c.dh, c.x, c.wg, c.wu, dx=torch.empty_like(c.x), trans_w=True)
    q = cb.gated_ffn_backward_query(d)
    assert q.split_k > 1 and q.workspace_bytes > q.workspace_min_bytes
    check_backward(cb, c, False, "f32", False, 0, "split", want_dw=False, want_h=False)
    whole, dx = torch.empty_like(c.x), torch.empty_like(c.x)
    cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=dx, trans_w=True)
    ws = torch.empty(q.workspace_min_bytes, dtype=torch.uint8, device="cuda")
    cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=whole, trans_w=True, workspace=ws)
    cb.sync_status()
    scale = dx.double().abs().max()
    assert ((whole.double() - dx.double()).abs() <= 2 * torch.finfo(torch.bfloat16).eps * scale).all()
    small = torch.empty(q.workspace_min_bytes - 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(cb.ChoreoError) as e:
        cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=whole, trans_w=True, workspace=small)
    assert e.value.code == cb.ERR_WORKSPACE


@pytest.mark.parametrize("act", ACTS)
def test_gradient_against_differences(cb, cuda, act):
    """The gradients' inner product with a direction equals the central
    difference of <H, dH> along it. Each of the inner product's terms is off by
    at most 3 half steps of bf16 (dG or dU, the output, and dH times act); over
    the 10^4 independent terms their sum stays far below a tenth of the sum of
    magnitudes. The difference's own error is of the order h^2 = 1e-8."""
    import torch
    c = Case(60, 72, 80, "bf16", act, False)
    if act == "relu":
        # keep G away from 0, where the slope jumps
        g = c.products()[0]
        c.dh[(g.abs() < 0.05)] = 0
    dx = torch.empty_like(c.x)
    dwg, dwu = torch.empty(80, 72, device="cuda"), torch.empty(80, 72, device="cuda")
    cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=dx, dw_gate=dwg, dw_up=dwu, act=act)
    cb.sync_status()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    x, dh = c.x.double(), c.dh.double()
    vx = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
    vg = torch.randn(dwg.shape, generator=gen, device="cuda", dtype=torch.float64) * 80 ** -0.5
    vu = torch.randn(dwu.shape, generator=gen, device="cuda", dtype=torch.float64) * 80 ** -0.5

    def value(t):
        return (act64((x + t * vx) @ (c.wgd + t * vg), act)[0] * ((x + t * vx) @ (c.wud + t * vu)) * dh).sum()

    h = 1e-4
    diff = (value(h) - value(-h)) / (2 * h)
    parts = [(dx.double(), vx), (dwg.double(), vg), (dwu.double(), vu)]
    inner = sum((a * b).sum() for a, b in parts)
    # |gradient| bounded through the magnitudes of its terms
    g, u, _, _ = c.products()
    v, dv = act64(g, act)
    adg, adu = (dh * u * dv).abs(), (dh * v).abs()
    mags = [(adg @ c.wgd.abs().t() + adu @ c.wud.abs().t()), x.abs().t() @ adg, x.abs().t() @ adu]
    bound = 3 * 2.0 ** -8 * sum((mag * b.abs()).sum() for mag, (_, b) in zip(mags, parts))
    assert abs(inner - diff) <= bound * 0.1 + 1e-3 * abs(diff), (inner.item(), diff.item(), bound.item())


def test_special_values(cb, cuda):
    """Large gates of either sign, and a NaN that stays in its row (forward,
    dX) and goes to its columns of the weight gradients."""
    import torch
    for m in (5, 200):   # both kernels
        for act in ACTS:
            c = Case(m, 136, 64, "bf16", act, False)
            c.x[0] *= 60.0
            h = torch.empty(m, 136, device="cuda", dtype=c.dt)
            cb.gated_ffn(c.x, c.wg, c.wu, h, act=act)
            g, u, eg, eu = c.products()
            want, e = c.hidden(g, u, eg, eu)
            assert_within(h, want, e + rounding(want.abs() + e, c.dt), (act, m))
            c.x[2, 7] = float("nan")
            ref = h.clone()
            cb.gated_ffn(c.x, c.wg, c.wu, h, act=act)
            cb.sync_status()
            rows = torch.arange(m, device="cuda") == 2
            assert torch.isnan(h[2]).all() and torch.equal(h[~rows], ref[~rows])


@pytest.mark.parametrize("m", [100, 300])
@pytest.mark.parametrize("trans", [False, True])
def test_offsets_past_32_bits(cb, cuda, m, trans):
    """Every matrix a column window of one buffer whose rows lie 2^23 elements
    apart: row 256 starts at 2^31."""
    import torch
    n, k, ld = 264, 296, 1 << 23
    c = Case(m, n, k, "bf16", "silu", trans)
    buf = torch.empty(300, ld, device="cuda", dtype=torch.bfloat16)
    used = [0]

    def window(rows, cols, src=None):
        v = buf[:rows, used[0]:used[0] + cols]
        used[0] += 512
        if src is not None:
            v.copy_(src)
        return v

    def far(src):
        return window(*src.shape, src)

    x, wg, wu, dh = far(c.x), far(c.wg), far(c.wu), far(c.dh)
    h, gate, up, dx = window(m, n), window(m, n), window(m, n), window(m, k)
    dwg, dwu = window(*wg.shape), window(*wg.shape)
    near = [torch.empty(*v.shape, device="cuda", dtype=torch.bfloat16) for v in (h, gate, up, dx, dwg, dwu)]
    cb.gated_ffn(x, wg, wu, h, trans_w=trans, gate=gate, up=up)
    cb.gated_ffn(c.x, c.wg, c.wu, near[0], trans_w=trans, gate=near[1], up=near[2])
    for kept in (False, True):
        cb.gated_ffn_backward(dh, x, wg, wu, dx=dx, dw_gate=dwg, dw_up=dwu, trans_w=trans,
                              **({"gate": gate, "up": up} if kept else {}))
        cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=near[3], dw_gate=near[4], dw_up=near[5], trans_w=trans,
                              **({"gate": near[1], "up": near[2]} if kept else {}))
        cb.sync_status()
        for got, want in zip((h, gate, up, dx, dwg, dwu), near):
            assert torch.equal(got, want)


def test_strides_shared_weight_matrix(cb, cuda):
    """Both weights as the halves of one matrix, and windows of larger x and h."""
    import torch
    m, n, k = 70, 128, 192
    w = matrix(k, 2 * n, torch.bfloat16, 1, k ** -0.5)
    big_x, big_h = matrix(m, k + 64, torch.bfloat16, 2), torch.zeros(m, n + 64, device="cuda", dtype=torch.bfloat16)
    x, h = big_x[:, 64:], big_h[:, 64:]
    cb.gated_ffn(x, w[:, :n], w[:, n:], h)
    flat = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    cb.gated_ffn(x.contiguous(), w[:, :n].contiguous(), w[:, n:].contiguous(), flat)
    cb.sync_status()
    assert torch.equal(h, flat) and (big_h[:, :64] == 0).all()


def test_repeats_bit_for_bit_on_streams_and_in_graphs(cb, cuda):
    """Two streams at once, each with its own workspace, and captured graphs."""
    import torch
    c = Case(300, 520, 264, "bf16", "silu", False)
    few = Case(9, 520, 264, "bf16", "silu", False)

    def outputs():
        return dict(dx=torch.empty_like(c.x.contiguous()), dw_gate=torch.empty(264, 520, device="cuda"),
                    dw_up=torch.empty(264, 520, device="cuda"), h=torch.empty(300, 520, device="cuda", dtype=c.dt))

    def work(o, ws, small):
        cb.gated_ffn(few.x, few.wg, few.wu, small)
        cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, workspace=ws, **o)

    need = cb.gated_ffn_backward_query(cb.ffn_grad_desc(c.dh, c.x, c.wg, c.wu, **outputs())).workspace_bytes
    ref, small_ref = outputs(), torch.empty(9, 520, device="cuda", dtype=c.dt)
    work(ref, torch.empty(need, dtype=torch.uint8, device="cuda"), small_ref)
    cb.sync_status()
    streams = [torch.cuda.Stream() for _ in range(2)]
    runs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        o, small = outputs(), torch.empty(9, 520, device="cuda", dtype=c.dt)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        with torch.cuda.stream(s):
            for _ in range(5):
                work(o, ws, small)
        runs.append((o, small, ws))
    torch.cuda.synchronize()
    graphs = []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        o, small = outputs(), torch.empty(9, 520, device="cuda", dtype=c.dt)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        with torch.cuda.graph(g, stream=s):
            work(o, ws, small)
        graphs.append((g, o, small, ws))
    for _ in range(3):
        for s, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    cb.sync_status()
    for o, small in [(r[0], r[1]) for r in runs] + [(g[1], g[2]) for g in graphs]:
        assert torch.equal(small, small_ref)
        for name in ref:
            assert torch.equal(o[name], ref[name]), name


def test_workspace_outlives_a_call_on_another_stream(cb, cuda):
    """The binding's own workspace (dG and dU, and repacked operands) is not
    handed to the current stream's allocations while a call on an explicit
    stream still uses it."""
    import torch
    c = Case(500, 1003, 331, "bf16", "silu", False, pads=(1, 1, 0))   # unaligned: repacks as well
    ref = torch.empty(500, 331, device="cuda", dtype=c.dt)
    cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=ref)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        outs = [torch.empty_like(ref) for _ in range(8)]
        torch.cuda.synchronize()
        for o in outs:
            cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=o, stream=stream)
            torch.empty(4 * 500 * 1008 * 2, dtype=torch.uint8, device="cuda").fill_(0x7F)  # current stream
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, ref)


def test_feed_forward_block_with_an_8_bit_down_projection(cb, cuda):
    """x -> gated_ffn -> quantize_block -> gemm_block_scaled with the residual
    as addend, for a prompt and for one token, against the 64-bit block. The
    e4m3 roundings (2^-4 of each value of h and of the down weight) dominate:
    their bound is that of the sum of magnitudes."""
    import torch
    n, k = 520, 264
    dt = torch.bfloat16
    wd = matrix(k, n, torch.float32, 9, n ** -0.5)
    kb, nb = -(-n // 128), -(-k // 128)
    qd = torch.empty(k, -(-n // 16) * 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :n]
    sd = torch.empty(kb, nb, device="cuda").t()
    cb.quantize_block(wd, qd, sd, block_rows=128)
    for m in (1, 33, 300):
        c = Case(m, n, k, "bf16", "silu", True, seed=m)
        h, y = torch.empty(m, n, device="cuda", dtype=dt), torch.empty(m, k, device="cuda", dtype=dt)
        qh = torch.empty(m, -(-n // 16) * 16, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :n]
        sh = torch.empty(kb, m, device="cuda").t()
        cb.gated_ffn(c.x, c.wg, c.wu, h, trans_w=True)
        cb.quantize_block(h, qh, sh)
        cb.gemm_block_scaled(qh, sh, qd, sd, y, beta=1.0, addend=c.x)
        cb.sync_status()
        g, u, eg, eu = c.products()
        hw, he = c.hidden(g, u, eg, eu)
        he = he + rounding(hw.abs() + he, dt)
        want = hw @ wd.double().t() + c.x.double()
        # e4m3: half a step of 2^-3 relative, and half of 2^-9 of the scale (amax / 448) below the normal range
        amax_h = (hw.abs() + he).amax()
        eh = he + 2.0 ** -4 * (hw.abs() + he) + 2.0 ** -10 * amax_h / 448
        ew = 2.0 ** -4 * wd.double().abs() + 2.0 ** -10 * wd.double().abs().amax() / 448
        e = eh @ (wd.double().abs() + ew).t() + (hw.abs() @ ew.t()) + 1e-5 * (hw.abs() @ wd.double().abs().t())
        assert_within(y, want, e + rounding(want.abs() + e, dt), m)
        # and close: the roundings are independent, so the errors add up like their root mean square
        rms = ((y.double() - want).square().mean().sqrt() / (want - c.x.double()).square().mean().sqrt()).item()
        assert rms < 0.1, rms
