"""The backward pass of the gated product against differences of the forward
formula, each gradient by itself and along its own sign pattern, where every
term counts with the same sign; and far out, with saturated gates, NaN and
infinities."""
from __future__ import annotations

import math

import pytest

from test_gated_ffn_gpu import ACTS, Case, act64, check_backward, rounding

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8   # half a step of bf16


def far_act64(g, act):
    """act64 with the normal distribution's lower tail through erfc: ndtr gives 0
    below -8 on the device."""
    import torch
    if act != "gelu":
        return act64(g, act)
    phi = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(60, 72, 80), (150, 200, 136)])
def test_each_gradient_against_differences(cb, cuda, act, trans, keep, m, n, k):
    """sum |gradient| equals the derivative of <H, dH> along the gradient's
    signs, taken as a central difference in 64 bits (step 1e-5: its own error is
    below 1e-7 of it).

    Tolerance. With d the direction, the sum is that of dG_ij a_ij + dU_ij b_ij,
    (a, b) = (d Wg, d Wu) for dX, (x d, 0) for dWg and (0, x d) for dWu. The
    independent errors are the roundings of dG, dU and dX to bf16, half a step
    of each, and with G and U kept in bf16 half a step of those through the
    formula (the slopes of the slopes are below 1.2). A sum of independent terms
    below e_i is beyond 6 sqrt(sum e_i^2) with a probability of 2 exp(-18)
    (Hoeffding). What may have one sign is the activation's 2^-16 and the fp32
    sums, less than 2^-15 of the sum of magnitudes."""
    import torch
    c = Case(m, n, k, "bf16", act, trans, seed=31)
    g, u, _, _ = c.products()
    if act == "relu":
        c.dh[g.abs() < 0.05] = 0   # the slope jumps at 0; G moves by less than 1e-5 * max_j sum_k |x| < 0.05
    shape = (n, k) if trans else (k, n)
    dx = torch.empty(m, k, device="cuda", dtype=c.dt)
    dwg, dwu = torch.empty(*shape, device="cuda"), torch.empty(*shape, device="cuda")
    kept = dict(gate=g.to(c.dt), up=u.to(c.dt)) if keep else {}
    cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=dx, dw_gate=dwg, dw_up=dwu, act=act, trans_w=trans, **kept)
    cb.sync_status()
    if trans:
        dwg, dwu = dwg.t(), dwu.t()
    x, dh = c.x.double(), c.dh.double()
    v, dv = act64(g, act)
    dg, du = dh * u * dv, dh * v
    eg, eu = HALF * dg.abs(), HALF * du.abs()
    if keep:
        eg = eg + HALF * dh.abs() * ((u * dv).abs() + 1.2 * (u * g).abs())
        eu = eu + HALF * dh.abs() * 1.2 * g.abs()

    def value(px, pg, pu):
        return (act64((x + px) @ (c.wgd + pg), act)[0] * ((x + px) @ (c.wud + pu)) * dh).sum()

    zero = torch.zeros((), device="cuda", dtype=torch.float64)
    t = 1e-5
    second = dh * u * (v / torch.where(g == 0, torch.ones_like(g), g))   # dG without its slope's second term
    for name, grad in (("dx", dx), ("dw_gate", dwg), ("dw_up", dwu)):
        grad = grad.double()
        d = torch.where(grad < 0, -1.0, 1.0).double()
        p = {"dx": (t * d, zero, zero), "dw_gate": (zero, t * d, zero), "dw_up": (zero, zero, t * d)}[name]
        diff = ((value(*p) - value(*[-q for q in p])) / (2 * t)).item()
        a = d @ c.wgd if name == "dx" else (x @ d if name == "dw_gate" else torch.zeros_like(g))
        b = d @ c.wud if name == "dx" else (x @ d if name == "dw_up" else torch.zeros_like(g))
        out = HALF * grad if name == "dx" else 2.0 ** -24 * grad
        rss = math.sqrt(((eg * a) ** 2).sum().item() + ((eu * b) ** 2).sum().item() + (out ** 2).sum().item())
        tol = 6 * rss + 2.0 ** -15 * ((dg * a).abs().sum() + (du * b).abs().sum()).item()
        got = (grad * d).sum().item()
        assert abs(got - diff) <= tol, (name, got, diff, tol)
        # the check tells a gradient from a wrong one
        assert tol < 0.02 * abs(diff), (name, tol, diff)
        if name == "dx":
            assert abs((dg * a).sum().item() - diff) > tol and abs((du * b).sum().item() - diff) > tol
        if name != "dw_up" and act != "relu":
            assert abs((second * a + du * b).sum().item() - diff) > tol, name


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [False, True])
def test_large_gates(cb, cuda, act, keep):
    """Gates of some hundred, of either sign: every output within its bounds."""
    for m, n, k in ((5, 136, 64), (200, 136, 64)):
        c = Case(m, n, k, "bf16", act, False, seed=3)
        c.x[0] *= 60.0
        check_backward(cb, c, keep, "f32", False, 0, (act, m))


def far_gates(dt):
    import torch
    mags = [0.0, 1e-6, 0.5, 5.0, 12.0, 20.0, 60.0, 86.0, 87.5, 88.5, 90.0, 104.0, 150.0, 1e3, 6e4]
    if dt == torch.bfloat16:
        mags += [1e-30, 1e10, 1e18, 1e20, 1e25, 1e30, 1e37, 3e38]
    g = torch.tensor(mags + [-x for x in mags], device="cuda", dtype=torch.float64).to(dt)
    assert torch.isfinite(g).all()
    return g


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("act", ACTS)
def test_saturated_kept_gates(cb, cuda, act, dt):
    """Kept gates up to the type's largest values, where the slopes are 0 or 1.
    With one weight the unit matrix and the other 0, dX is dG or dU itself.

    Relative errors: the exponent is below 104 where the result is not 0, off by
    four roundings of 2^-24 of it, and __expf by 2 + 1.2 * 104 units of 2^-23:
    less than 1e-4 in all. Below 2^-120 the divisions may give 0."""
    import torch
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dt]
    gates = far_gates(t)
    m, n = 37, 64
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    gate = gates[torch.arange(m * n, device="cuda") % gates.numel()].view(m, n).contiguous()
    up = (0.25 + 0.7 * torch.rand(m, n, generator=gen, device="cuda")).to(t)
    dh = (torch.rand(m, n, generator=gen, device="cuda") - 0.5).to(t)
    x = torch.randn(m, n, generator=gen, device="cuda").to(t)
    eye, none = torch.eye(n, device="cuda", dtype=t), torch.zeros(n, n, device="cuda", dtype=t)
    dg, du, h = (torch.empty(m, n, device="cuda", dtype=t) for _ in range(3))
    cb.gated_ffn_backward(dh, x, eye, none, dx=dg, gate=gate, up=up, h=h, act=act)
    cb.gated_ffn_backward(dh, x, none, eye, dx=du, gate=gate, up=up, act=act)
    cb.sync_status()
    g, u, d = gate.double(), up.double(), dh.double()
    v, dv = far_act64(g, act)
    share = torch.where(g == 0, torch.zeros_like(g), v / torch.where(g == 0, torch.ones_like(g), g))
    ev = 1e-4 * v.abs() + 2.0 ** -120 * g.abs().clamp_min(1)
    edv = 1e-4 * (dv.abs() + (dv - share).abs() + share.abs()) + 2.0 ** -120 * (1 + g.square().clamp_max(2e4))
    for name, got, want, e in (("dg", dg, d * u * dv, (d * u).abs() * edv), ("du", du, d * v, d.abs() * ev),
                               ("h", h, v * u, ev * u.abs())):
        off = (got.double() - want).abs()
        bound = e + rounding(want.abs() + e, t)
        worst = (off / bound).max().item()
        assert torch.isfinite(got).all() and (off <= bound).all(), (name, worst, g.flatten()[(off / bound).argmax()])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("m", [5, 200])
def test_nan_and_infinity_stay_in_their_row_and_column(cb, cuda, act, keep, m):
    """A NaN in dH reaches its row of dX and its column of both weight
    gradients and nothing else; so does an infinity, as a value that is not
    finite or as a 0 (or NaN) where it meets a 0."""
    import torch
    n, k = 136, 64
    c = Case(m, n, k, "bf16", act, False, seed=5)
    gate = up = None
    if keep:
        g, u, _, _ = c.products()
        gate, up = g.to(c.dt), u.to(c.dt)

    def run():
        dx = torch.empty(m, k, device="cuda", dtype=c.dt)
        dwg, dwu = torch.empty(k, n, device="cuda"), torch.empty(k, n, device="cuda")
        cb.gated_ffn_backward(c.dh, c.x, c.wg, c.wu, dx=dx, dw_gate=dwg, dw_up=dwu, gate=gate, up=up, act=act)
        cb.sync_status()
        return dx, dwg, dwu

    ref = run()
    rows, cols = torch.arange(m, device="cuda") != 2, torch.arange(n, device="cuda") != 9
    for bad in (float("nan"), float("inf")):
        c.dh[2, 9] = bad
        dx, dwg, dwu = run()
        assert torch.equal(dx[rows], ref[0][rows])
        assert torch.equal(dwg[:, cols], ref[1][:, cols]) and torch.equal(dwu[:, cols], ref[2][:, cols])
        if bad != bad:
            assert torch.isnan(dx[2]).all() and torch.isnan(dwg[:, 9]).all() and torch.isnan(dwu[:, 9]).all()
        elif act != "relu":
            assert not torch.isfinite(dx[2]).any()
    if keep:   # x then only enters the weight gradients: row 7 of them
        c.dh[2, 9] = 0.0
        c.x[2, 7] = float("nan")
        ref0 = run()
        rest = torch.arange(k, device="cuda") != 7
        c.x[2, 7] = 0.0
        ref1 = run()
        assert torch.equal(ref0[0], ref1[0])
        for a, b in zip(ref0[1:], ref1[1:]):
            assert torch.isnan(a[7]).all() and torch.equal(a[rest], b[rest])
    else:      # and here G, U and with them the whole row of dX and both weight gradients
        c.dh[2, 9] = 0.5
        c.x[2, 7] = float("nan")
        dx, dwg, dwu = run()
        assert torch.isnan(dx[2]).all() and torch.equal(dx[rows], ref[0][rows])
        assert torch.isnan(dwg).all() and torch.isnan(dwu).all()
