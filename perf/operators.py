"""Measured cases of the large-language-model operators: the gated feed-forward
product and its backward pass, the block quantiser and the 8-bit block-scaled
matrix product.

`own` chooses between the operators' plain form in elementary torch operations
and this repository's kernels; everything else is the same for both."""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_F8 = torch.float8_e4m3fn
_TINY = 2.0 ** -100  # floor of a block's largest magnitude


def _factors(amax):
    """448 / amax and amax / 448, each rounded once (a Python number on one side would make torch
    multiply by a rounded reciprocal)."""
    top = torch.full_like(amax, 448.0)
    return top / amax, amax / top


def _package():
    """This repository's package (its folder name has a hyphen)."""
    if "choreo_b200" not in sys.modules:
        path = Path(__file__).resolve().parents[1] / "choreo-ir_b200" / "__init__.py"
        spec = importlib.util.spec_from_file_location("choreo_b200", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["choreo_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["choreo_b200"]


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decoder: latency, bound by reading both weights once
        {"name": "gate-one-token", "op": "gate", "m": 1, "k": 4096, "n": 10240, "dt": "bf16", "act": "silu",
         "trans": True, "save": False},
        # a ragged decode batch, odd hidden width, weights stored k x n
        {"name": "gate-batch-ragged", "op": "gate", "m": 77, "k": 2056, "n": 5461, "dt": "f16", "act": "gelu_tanh",
         "trans": False, "save": False},
        # a training forward over a long batch, keeping gate and up for the backward pass
        {"name": "gate-train", "op": "gate", "m": 8192, "k": 4096, "n": 10240, "dt": "bf16", "act": "silu",
         "trans": False, "save": True},
        # backward pass of a mid-size block from the kept gate and up
        {"name": "grad-kept", "op": "grad", "m": 2049, "k": 2048, "n": 5632, "dt": "f16", "act": "gelu",
         "trans": True, "keep": True},
        # backward pass that computes gate and up again (and h, for the down projection's gradient)
        {"name": "grad-again", "op": "grad", "m": 8192, "k": 4096, "n": 10240, "dt": "bf16", "act": "silu",
         "trans": False, "keep": False},
        # the activations of a few decode tokens: latency
        {"name": "quant-tokens", "op": "quant", "rows": 13, "cols": 4096, "dt": "bf16", "block": 1, "transpose": False},
        # the activations of a long batch before an 8-bit product: bandwidth
        {"name": "quant-batch", "op": "quant", "rows": 8192, "cols": 10240, "dt": "bf16", "block": 1,
         "transpose": False},
        # an odd-sized f32 master weight, its transpose in 128 x 128 blocks (for the input gradient)
        {"name": "quant-weight-transposed", "op": "quant", "rows": 8191, "cols": 4100, "dt": "f32", "block": 128,
         "transpose": True},
        # a down projection of a small decode batch: bound by reading the weight once
        {"name": "block-decode", "op": "block", "m": 16, "n": 4096, "k": 10240, "c": "bf16", "b_block": 128,
         "accumulate": False},
        # odd sizes that end inside tiles and inside a scale block
        {"name": "block-ragged", "op": "block", "m": 1031, "n": 2053, "k": 1999, "c": "f16", "b_block": 128,
         "accumulate": False},
        # a large prefill or training forward product
        {"name": "block-large", "op": "block", "m": 8192, "n": 8192, "k": 8192, "c": "bf16", "b_block": 128,
         "accumulate": False},
        # a weight gradient added to the f32 sum so far: both operands in 1 x 128 blocks along the tokens
        {"name": "block-weight-grad", "op": "block", "m": 4096, "n": 10240, "k": 8192, "c": "f32", "b_block": 1,
         "accumulate": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gate", "grad", "quant", "block"])
    dt = rng.choice(["bf16", "f16"])
    act = rng.choice(["silu", "gelu", "gelu_tanh", "relu"])
    if op in ("gate", "grad"):
        m = _log(rng, 1, 8192) if op == "gate" else _log(rng, 16, 8192)
        k, n = 8 * _log(rng, 32, 1024), _log(rng, 200, 12288)
        while m * k * n > 8192 * 4096 * 10240:
            m = (m + 1) // 2
        case = {"op": op, "m": m, "k": k, "n": n, "dt": dt, "act": act, "trans": rng.random() < 0.5}
        case["save" if op == "gate" else "keep"] = rng.random() < 0.5
        return case
    if op == "quant":
        rows, cols = _log(rng, 1, 16384), _log(rng, 100, 16384)
        while rows * cols > 8192 * 10240:
            rows = (rows + 1) // 2
        return {"op": op, "rows": rows, "cols": cols, "dt": rng.choice(["bf16", "f16", "f32"]),
                "block": rng.choice([1, 128]), "transpose": rng.random() < 0.5}
    m, n, k = _log(rng, 1, 8192), _log(rng, 128, 12288), _log(rng, 128, 12288)
    while m * n * k > 8192 ** 3:
        m = (m + 1) // 2
    return {"op": op, "m": m, "n": n, "k": k, "c": rng.choice(["bf16", "f16", "f32"]),
            "b_block": rng.choice([1, 128]), "accumulate": rng.random() < 0.3}


# --------------------------------------------------------------------- inputs
def _rows(shape, dtype, multiple=8):
    """A matrix whose rows start on 16-byte boundaries, as a program that owns it lays it out."""
    pad = -(-shape[1] // multiple) * multiple
    return torch.empty(shape[0], pad, dtype=dtype, device="cuda")[:, : shape[1]]


def _normal(gen, shape, std, dtype):
    out = _rows(shape, dtype, 16 // torch.empty(0, dtype=dtype).element_size())
    return out.copy_(torch.randn(shape, generator=gen, device="cuda").mul_(std))


def _activations(gen, rows, cols):
    """Token activations: a normal bulk with a few channels that stand out."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def _to_blocks(x, block):
    """e4m3 values and scales of x in block x 128 blocks: what a program has before an 8-bit product."""
    rows, cols = x.shape
    kb, rb = -(-cols // 128), -(-rows // block)
    full = torch.zeros(rb * block, kb * 128, device="cuda")
    full[:rows, :cols] = x
    parts = full.view(rb, block, kb, 128)
    amax = parts.abs().amax(dim=(1, 3)).clamp_min(_TINY)
    factor, scales = _factors(amax)
    q8 = (parts * factor[:, None, :, None]).reshape(full.shape)[:rows, :cols].to(_F8)
    q = _rows((rows, cols), torch.uint8, 16)
    q.copy_(q8.view(torch.uint8))
    scale = torch.empty(kb, rb, device="cuda").t()  # the rows of one k-block next to each other
    scale.copy_(scales)
    return q.view(_F8), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] in ("gate", "grad"):
        m, n, k, dt = case["m"], case["n"], case["k"], _DT[case["dt"]]
        s["x"] = _normal(gen, (m, k), 1.0, dt)
        shape = (n, k) if case["trans"] else (k, n)
        s["w_gate"] = _normal(gen, shape, k ** -0.5, dt)
        s["w_up"] = _normal(gen, shape, k ** -0.5, dt)
        if case["op"] == "gate":
            s["h"] = _rows((m, n), dt)
            s["gate"] = _rows((m, n), dt) if case["save"] else None
            s["up"] = _rows((m, n), dt) if case["save"] else None
        else:
            s["dh"] = _normal(gen, (m, n), 0.1, dt)
            s["gate"] = _normal(gen, (m, n), 1.0, dt) if case["keep"] else None
            s["up"] = _normal(gen, (m, n), 1.0, dt) if case["keep"] else None
            s["h"] = None if case["keep"] else _rows((m, n), dt)
            s["dx"] = _rows((m, k), dt)
            s["dw_gate"], s["dw_up"] = _rows(shape, dt), _rows(shape, dt)
    elif case["op"] == "quant":
        rows, cols = case["rows"], case["cols"]
        x = _rows((rows, cols), _DT[case["dt"]], 8)
        s["x"] = x.copy_(_activations(gen, rows, cols))
        r, c = (cols, rows) if case["transpose"] else (rows, cols)
        s["q"] = _rows((r, c), torch.uint8, 16).view(_F8)
        s["scale"] = torch.empty(-(-c // 128), -(-r // case["block"]), device="cuda").t()
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["scale_a"] = _to_blocks(_activations(gen, m, k), 1)
        s["b"], s["scale_b"] = _to_blocks(torch.randn(n, k, generator=gen, device="cuda").mul_(k ** -0.5),
                                          case["b_block"])
        dt = _DT[case["c"]]
        s["c"] = _rows((m, n), dt, 8)
        s["c0"] = _normal(gen, (m, n), 1.0, dt) if case["accumulate"] else None
    return s


# --------------------------------------------------------------- plain form
def _act(g, act):
    """The activation and its derivative, elementwise."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * g * g)
    on = (g > 0).to(g.dtype)
    return g * on, on


def _plain_gate(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    if case["trans"]:
        wg, wu = wg.t(), wu.t()
    g, u = x @ wg, x @ wu
    out = {"h": (_act(g, case["act"])[0] * u).to(dt)}
    if case["save"]:
        out["gate"], out["up"] = g.to(dt), u.to(dt)
    return out


def _plain_grad(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, dh = s["x"].float(), s["w_gate"].float(), s["w_up"].float(), s["dh"].float()
    if case["trans"]:
        wg, wu = wg.t(), wu.t()
    g, u = (s["gate"].float(), s["up"].float()) if case["keep"] else (x @ wg, x @ wu)
    value, slope = _act(g, case["act"])
    dg, du = dh * u * slope, dh * value
    out = {"dx": (dg @ wg.t() + du @ wu.t()).to(dt)}
    dwg, dwu = x.t() @ dg, x.t() @ du
    out["dw_gate"], out["dw_up"] = (dwg.t().to(dt), dwu.t().to(dt)) if case["trans"] else (dwg.to(dt), dwu.to(dt))
    if not case["keep"]:
        out["h"] = (value * u).to(dt)
    return out


def _plain_quant(s):
    case = s["case"]
    x = s["x"].float()
    if case["transpose"]:
        x = x.t()
    rows, cols = x.shape
    block = case["block"]
    kb, rb = -(-cols // 128), -(-rows // block)
    full = torch.zeros(rb * block, kb * 128, device=x.device)
    full[:rows, :cols] = x
    parts = full.view(rb, block, kb, 128)
    amax = parts.abs().amax(dim=(1, 3)).clamp_min(_TINY)
    factor, scale = _factors(amax)
    q = (parts * factor[:, None, :, None]).reshape(full.shape)[:rows, :cols]
    return {"q": q.to(_F8), "scale": scale}


def _plain_block(s):
    case, c = s["case"], s["c"]
    m, n, k = case["m"], case["n"], case["k"]
    sa = s["scale_a"].repeat_interleave(128, 1)[:, :k]
    sb = s["scale_b"].repeat_interleave(128, 1)[:, :k]
    if case["b_block"] == 128:
        sb = sb.repeat_interleave(128, 0)[:n]
    out = (s["a"].float() * sa) @ (s["b"].float() * sb).t()
    if case["accumulate"]:
        out = out + s["c0"].float()
    return {"c": out.to(c.dtype)}


# ------------------------------------------------------------ the framework's
def _own_gate(s):
    cb, case = _package(), s["case"]
    cb.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["h"], act=case["act"], trans_w=case["trans"], gate=s["gate"],
                 up=s["up"])
    return {k: s[k] for k in ("h", "gate", "up") if s[k] is not None}


def _own_grad(s):
    cb, case = _package(), s["case"]
    cb.gated_ffn_backward(s["dh"], s["x"], s["w_gate"], s["w_up"], dx=s["dx"], dw_gate=s["dw_gate"],
                          dw_up=s["dw_up"], gate=s["gate"], up=s["up"], h=s["h"], act=case["act"],
                          trans_w=case["trans"])
    return {k: s[k] for k in ("dx", "dw_gate", "dw_up", "h") if s[k] is not None}


def _own_quant(s):
    cb, case = _package(), s["case"]
    cb.quantize_block(s["x"], s["q"], s["scale"], block_rows=case["block"], transpose=case["transpose"])
    return {"q": s["q"], "scale": s["scale"]}


def _own_block(s):
    cb, case = _package(), s["case"]
    cb.gemm_block_scaled(s["a"], s["scale_a"], s["b"], s["scale_b"], s["c"], beta=1.0 if case["accumulate"] else 0.0,
                         addend=s["c0"])
    return {"c": s["c"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"gate": _own_gate, "grad": _own_grad, "quant": _own_quant, "block": _own_block}[op](state)
    return {"gate": _plain_gate, "grad": _plain_grad, "quant": _plain_quant, "block": _plain_block}[op](state)


def work(case):
    if case["op"] in ("gate", "grad"):
        m, n, k = case["m"], case["n"], case["k"]
        if case["op"] == "gate":
            return {"bytes": 2 * (m * k + 2 * k * n + m * n * (3 if case["save"] else 1)), "flops": 4 * m * n * k}
        # read x, dh, both weights (and gate, up); write dx, both weight gradients (and h)
        return {"bytes": 2 * (2 * m * k + 4 * k * n + m * n * (3 if case["keep"] else 2)),
                "flops": (8 if case["keep"] else 12) * m * n * k}
    if case["op"] == "quant":
        r, c = (case["cols"], case["rows"]) if case["transpose"] else (case["rows"], case["cols"])
        scales = -(-r // case["block"]) * -(-c // 128)
        return {"bytes": r * c * (5 if case["dt"] == "f32" else 3) + 4 * scales, "flops": 2 * r * c}
    m, n, k = case["m"], case["n"], case["k"]
    kb = -(-k // 128)
    size = 4 if case["c"] == "f32" else 2
    return {"bytes": m * k + n * k + 4 * kb * (m + -(-n // case["b_block"]))
            + m * n * size * (2 if case["accumulate"] else 1), "flops": 2 * m * n * k}


# ------------------------------------------------------------ 64-bit values
def _phi(z):
    return torch.special.ndtr(z)


def _exact_act(z, act):
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        return z * _phi(z), _phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        inner = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p = torch.sigmoid(2 * inner)  # (1 + tanh(inner)) / 2
        slope = 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z ** 2)
        return z * p, p + z * p * (1 - p) * slope
    return torch.relu(z), torch.where(z > 0, 1.0, 0.0).double()


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.dtype != _F8}
    if case["op"] in ("gate", "grad"):
        eq = "mk,nk->mn" if case["trans"] else "mk,kn->mn"
        if case["op"] == "gate":
            g, u = torch.einsum(eq, d["x"], d["w_gate"]), torch.einsum(eq, d["x"], d["w_up"])
            out = {"h": _exact_act(g, case["act"])[0] * u}
            return {**out, "gate": g, "up": u} if case["save"] else out
        if case["keep"]:
            g, u = d["gate"], d["up"]
        else:
            g, u = torch.einsum(eq, d["x"], d["w_gate"]), torch.einsum(eq, d["x"], d["w_up"])
        v, dv = _exact_act(g, case["act"])
        pg, pu = d["dh"] * u * dv, d["dh"] * v
        back = "mn,nk->mk" if case["trans"] else "mn,kn->mk"
        wgrad = "mn,mk->nk" if case["trans"] else "mn,mk->kn"
        out = {"dx": torch.einsum(back, pg, d["w_gate"]) + torch.einsum(back, pu, d["w_up"]),
               "dw_gate": torch.einsum(wgrad, pg, d["x"]), "dw_up": torch.einsum(wgrad, pu, d["x"])}
        return out if case["keep"] else {**out, "h": v * u}
    if case["op"] == "quant":
        z = d["x"].t() if case["transpose"] else d["x"]
        r, c = z.shape
        top = z.abs()
        top = torch.nn.functional.pad(top, (0, -c % 128, 0, -r % case["block"]))
        top = top.unflatten(1, (-1, 128)).amax(2).unflatten(0, (-1, case["block"])).amax(1).clamp(min=_TINY)
        # the factor 448 / top and the product with it are 32-bit numbers by definition (the product is
        # exact in 64 bits): many products lie on or next to the middle of two e4m3 values
        factor = (torch.full_like(top, 448.0) / top).float().double()
        v = z * factor.repeat_interleave(case["block"], 0)[:r].repeat_interleave(128, 1)[:, :c]
        v = v.float().double()
        # nearest e4m3, ties to even: 4 significant bits, steps of 2^-9 below 2^-6
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        return {"q": torch.round(v / step) * step, "scale": top / 448.0}
    sums = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
    if case["accumulate"]:
        sums += d["c0"]
    for j in range(0, case["n"], 128):  # columns of one scale block at a time
        bj = s["b"][j:j + 128].to(torch.float32).double()
        sj = d["scale_b"][j:j + 128] if case["b_block"] == 1 else d["scale_b"][j // 128][None]
        bj = bj * sj.repeat_interleave(128, 1)[:, :case["k"]]
        if j == 0:
            wide = s["a"].to(torch.float32).double() * d["scale_a"].repeat_interleave(128, 1)[:, :case["k"]]
        sums[:, j:j + 128] += wide @ bj.t()
    return {"c": sums}
