"""Refusals of the gated feed-forward, quantisation and block-scaled calls that
need no GPU: every contract is checked before the first CUDA call, with a code
and a message, and the bindings' own checks of shapes and types."""
from __future__ import annotations

import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "choreo_b200.h"


def test_struct_layout_matches_c_compiler(cb, tmp_path):
    structs = {"choreo_ffn_desc": cb.FfnDesc, "choreo_ffn_grad_desc": cb.FfnGradDesc,
               "choreo_quant_desc": cb.QuantDesc, "choreo_gemm_block_desc": cb.GemmBlockDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0; }"]))
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    got = {}
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            s, f, v = line.split()
            got[(s, f)] = int(v)
    for name, py in structs.items():
        assert got[(name, "size")] == C.sizeof(py), name
        for f, _ in py._fields_:
            assert got[(name, f)] == getattr(py, f).offset, (name, f)


def refused(cb, fn, desc, code, message):
    rc = fn(desc)
    text = cb.lib.choreo_last_error().decode()
    assert rc == code and message in text, (rc, text)


def _fill(d, **kw):
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def ffn(cb, **kw):
    d = _fill(cb.FfnDesc(), m=64, n=96, k=32, dtype=cb.BF16, act=0, x=0x1000, ldx=32, w_gate=0x2000, w_up=0x3000,
              ldw=96, trans_w=0, h=0x4000, ldh=96)
    return _fill(d, **kw)


FFN = [
    (dict(m=0), -1, "Invalid dimensions"), (dict(n=-1), -1, "Invalid dimensions"), (dict(k=0), -1, "Invalid dimensions"),
    (dict(m=1 << 31), -2, "2^30-1"), (dict(n=1 << 30, ldw=1 << 30, ldh=1 << 30), -2, "2^29-1"),
    (dict(dtype=9), -2, "not f16 or bf16"), (dict(act=4), -2, "unknown activation"), (dict(act=-1), -2, "unknown activation"),
    (dict(x=None), -1, "X has null"), (dict(w_gate=None), -1, "weight has null"), (dict(w_up=None), -1, "weight has null"),
    (dict(ldx=31), -1, "ldx=31"), (dict(ldw=95), -1, "ldw=95"), (dict(trans_w=1, ldw=31), -1, "ldw=31"),
]


@pytest.mark.parametrize("kw,code,msg", FFN + [
    (dict(h=None), -1, "H has null"), (dict(ldh=95), -1, "ldh=95"),
    (dict(gate=0x5000), -1, "kept together"), (dict(up=0x5000), -1, "kept together"),
    (dict(gate=0x5000, up=0x6000, ld_gu=3), -1, "ld_gu=3"),
])
def test_forward_refusals(cb, kw, code, msg):
    d = ffn(cb, **kw)
    refused(cb, lambda x: cb.lib.choreo_gated_ffn(C.byref(x), None, 0, None), d, code, msg)
    out = cb.LaunchConfig()
    refused(cb, lambda x: cb.lib.choreo_gated_ffn_query(C.byref(x), C.byref(out)), d, code, msg)


def grad(cb, **kw):
    d = _fill(cb.FfnGradDesc(), m=64, n=96, k=32, dtype=cb.BF16, act=0, x=0x1000, ldx=32, w_gate=0x2000, w_up=0x3000,
              ldw=96, trans_w=0, dtype_dw=cb.F32, dh=0x4000, ld_dh=96, dx=0x5000, ld_dx=32, dw_gate=0x6000,
              dw_up=0x7000, ld_dw=96)
    return _fill(d, **kw)


@pytest.mark.parametrize("kw,code,msg", FFN + [
    (dict(dh=None), -1, "dH has null"), (dict(ld_dh=95), -1, "ld_dh=95"),
    (dict(gate=0x8000), -1, "kept together"), (dict(gate=0x8000, up=0x9000, ld_gu=95), -1, "ld_gu=95"),
    (dict(dw_up=None), -1, "computed together"), (dict(dx=None, dw_gate=None, dw_up=None), -1, "neither dX"),
    (dict(ld_dx=31), -1, "ld_dx=31"), (dict(ld_dw=95), -1, "ld_dw=95"), (dict(dtype_dw=8), -2, "dtype_dw 8"),
    (dict(h=0xA000, ldh=1), -1, "ldh=1"),
])
def test_backward_refusals(cb, kw, code, msg):
    d = grad(cb, **kw)
    refused(cb, lambda x: cb.lib.choreo_gated_ffn_backward(C.byref(x), None, 0, None), d, code, msg)
    out = cb.LaunchConfig()
    refused(cb, lambda x: cb.lib.choreo_gated_ffn_backward_query(C.byref(x), C.byref(out)), d, code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=-1), -1, "negative size"), (dict(dtype=3), -2, "unsupported dtype"),
    (dict(block_rows=64), -2, "neither 1 nor 128"), (dict(rows=1 << 31), -2, "2^31-1"),
    (dict(x=None), -1, "null data pointer"), (dict(q=None), -1, "null data pointer"),
    (dict(scale=None), -1, "null data pointer"), (dict(ldx=299), -1, "ldx=299"), (dict(ldq=299), -1, "ldq=299"),
    (dict(transpose=1, ldq=199), -1, "ldq=199"), (dict(scale_row=0), -1, "must be positive"),
    (dict(scale_blk=-1), -1, "must be positive"),
])
def test_quantize_refusals(cb, kw, code, msg):
    d = _fill(cb.QuantDesc(), rows=200, cols=300, dtype=cb.BF16, x=0x1000, ldx=300, block_rows=1, q=0x2000, ldq=300,
              scale=0x3000, scale_row=1, scale_blk=200)
    refused(cb, lambda x: cb.lib.choreo_quantize_block(C.byref(x), None), _fill(d, **kw), code, msg)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(m=0), -1, "Invalid matrix dimensions"), (dict(k=-5), -1, "Invalid matrix dimensions"),
    (dict(n=1 << 31), -2, "2^30-1"), (dict(a=None), -1, "operand has null"), (dict(scale_b=None), -1, "scale has null"),
    (dict(c=None), -1, "Output tensor C"), (dict(dtype_c=3), -2, "unsupported output"),
    (dict(block_b=64), -2, "neither 1 nor 128"), (dict(lda=176), -1, "smaller than K"),
    (dict(lda=193), -1, "multiples of 16"), (dict(ldb=200), -1, "multiples of 16"), (dict(a=0x1008), -1, "multiples of 16"),
    (dict(b=0x2001), -1, "multiples of 16"), (dict(ldc=9), -1, "ldc=9"), (dict(scale_a_blk=-1), -1, "negative scale"),
    (dict(addend=0x7000, ld_addend=3), -1, "ld_addend=3"), (dict(bias=0x8000, dtype_bias=2), -2, "bias dtype"),
])
def test_block_scaled_refusals(cb, kw, code, msg):
    d = _fill(cb.GemmBlockDesc(), m=100, n=40, k=180, a=0x1000, lda=192, scale_a=0x3000, scale_a_row=1, scale_a_blk=100,
              b=0x2000, ldb=192, scale_b=0x4000, scale_b_row=1, scale_b_blk=1, block_b=128, dtype_c=cb.BF16, c=0x5000,
              ldc=40, alpha=1.0)
    d = _fill(d, **kw)
    refused(cb, lambda x: cb.lib.choreo_gemm_block_scaled(C.byref(x), None), d, code, msg)
    out = cb.LaunchConfig()
    refused(cb, lambda x: cb.lib.choreo_gemm_block_scaled_query(C.byref(x), C.byref(out)), d, code, msg)


def test_null_descriptors(cb):
    for fn in (lambda: cb.lib.choreo_gated_ffn(None, None, 0, None),
               lambda: cb.lib.choreo_gated_ffn_backward(None, None, 0, None),
               lambda: cb.lib.choreo_quantize_block(None, None), lambda: cb.lib.choreo_gemm_block_scaled(None, None)):
        assert fn() == cb.ERR_INVALID_ARG and "null descriptor" in cb.lib.choreo_last_error().decode()


def test_host_memory_is_refused(cb):
    """Pointers that are no device memory never reach a launch (here there is no
    CUDA device at all: the look-up itself fails, with the same code)."""
    d = ffn(cb)
    assert cb.lib.choreo_gated_ffn(C.byref(d), None, 0, None) == cb.ERR_INVALID_ARG


def test_binding_checks_shapes_and_types(cb):
    import torch
    x, w, h = torch.zeros(4, 8).bfloat16(), torch.zeros(8, 6).bfloat16(), torch.zeros(4, 6).bfloat16()
    q, c = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 4)
    cases = [
        lambda: cb.gated_ffn(x, w, w, torch.zeros(4, 5).bfloat16(), stream=0),
        lambda: cb.gated_ffn(x, w, w.half(), h, stream=0),
        lambda: cb.gated_ffn(x, w, torch.zeros(8, 7).bfloat16()[:, :6], h, stream=0),
        lambda: cb.gated_ffn(x, w.t().contiguous().t(), w, h, stream=0),
        lambda: cb.gated_ffn(x, w, w, h, act="tanh", stream=0),
        lambda: cb.gated_ffn(x, w, w, h, gate=h, up=torch.zeros(4, 7).bfloat16()[:, :6], stream=0),
        lambda: cb.gated_ffn_backward(h, x, w, w, dx=torch.zeros(4, 9).bfloat16(), stream=0),
        lambda: cb.gated_ffn_backward(h, x, w, w, dw_gate=w.float(), dw_up=w, stream=0),
        lambda: cb.quantize_block(x, torch.zeros(4, 8), torch.zeros(4, 1), stream=0),
        lambda: cb.quantize_block(x, torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(1, 1), stream=0),
        lambda: cb.quantize_block(x, torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4, 1), transpose=True, stream=0),
        lambda: cb.gemm_block_scaled(x, torch.zeros(4, 1), x, torch.zeros(1, 1), h, stream=0),
        lambda: cb.gemm_block_scaled(q, torch.zeros(4, 1), q, torch.zeros(4, 1), c, bias=torch.zeros(3), stream=0),
        lambda: cb.gemm_block_scaled(q, torch.zeros(4, 1), q, torch.zeros(4, 1), c, bias=torch.zeros(8)[::2], stream=0),
    ]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"case {i} was accepted")
